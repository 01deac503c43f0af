// Writing the paged key / value cache: per-head RMS norm of queries and keys,
// position rotation, and the append of keys and values in bf16 or 4 bits, in
// one pass over the rows of a fused projection; and reading it back as values.
//
// Per head x[hd] of a row at position p: y = x * rsqrt(sum x^2 / hd + eps) * g
// (queries and keys, where there is a g); (y_a, y_b) -> (y_a cos - y_b sin,
// y_b cos + y_a sin) over the rotated pairs; then one rounding: bf16, or per 64
// dimensions m = bf16(min), s = bf16((max - min) * r), r = 1 / 15 rounded to f32
// (a product in place of a division; the two differ where (max - min) / 15 lies
// within 2^-23 of it from a tie of bf16), code = round((y - m) / s) clamped to 0..15.  The codes are taken against the rounded m and s, so
// their rounding does not add to the value's error except at the ends.
//
// A thread holds 8 neighbouring dimensions in f32 (one 16-byte load of bf16,
// two of f32), a head is hd / 8 neighbouring lanes: the norm's sum, the
// half-apart rotation partner and the group's extremes are shuffles within
// them, so nothing passes through shared memory.  A warp stays with one row and
// keeps its rotation, page and norm weights in registers while it walks over the
// heads, the next head's load under way.
//
// What bounds it: for many rows memory and issue about alike (16384 rows of 16 +
// 2 x 16 heads of 128, bf16: 91 us, 4.5 TB/s read and written, 151 instructions a
// warp and step at 64 % of the issue slots; a second step's load under way
// changes nothing), in 4 bits issue (4093 rows of 28 + 2 x 4 heads: 27 us under
// the profiler, 70 % of the slots), for few the latency of seq -> page -> store.
#include "paged.cuh"

using namespace sm100;

namespace {

constexpr int kAppendWarps = 148 * 16;   // enough to keep the GPU's memory busy

struct AppendParams {
  const void *qkv;
  const float *g_q, *g_k, *cos_t, *sin_t;
  const int32_t *pos, *seq;
  __nv_bfloat16 *q_out;
  int64_t ld;
  int T, heads, rot, n_pos, pairs;
  int parts, steps;   // warps of a row, and a warp's steps
  float eps;
};

__device__ __forceinline__ void load8(const float *p, float x[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// 8 values as they were loaded
template <typename In>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void get(float x[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
  }
};
template <>
struct Raw<float> {
  float4 a, b;
  __device__ __forceinline__ void get(float x[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
__device__ __forceinline__ Raw<__nv_bfloat16> load_raw(const __nv_bfloat16 *p) { return {ld_stream_u4(p)}; }
__device__ __forceinline__ Raw<float> load_raw(const float *p) { return {ld_stream_f4(p), ld_stream_f4(p + 4)}; }

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ uint4 pack8(const float x[8]) {
  return make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
}

// min / max that keep a NaN (a group with one must not read as numbers)
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float shfl_add(float v, int o) { return __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o)); }

// sum x^2 of a head in one fixed order for each head size, each step rounded on
// its own: 256 dimensions add their two halves, 128 add up runs of 4 neighbours,
// and what there is adds its halves, element i with i + n / 2, until one is left.
// There is no numerical reason for these orders, and they are not the cheapest:
// the formula written in torch operations is summed like this on this GPU, and a
// key gets the code here that it gets there, ties between two codes included.
template <int HD>
__device__ __forceinline__ float sum_squares(const float x[8]) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; i++) s[i] = __fmul_rn(x[i], x[i]);
  if constexpr (HD == 64) {   // unit 1: 32, 16 and 8 apart are lanes, 4, 2 and 1 apart within the lane
    const int hl = threadIdx.x & 7;
    float a[4], b[2];
#pragma unroll
    for (int i = 0; i < 4; i++) {   // each exchange halves what a lane holds
      const float got = __shfl_xor_sync(0xffffffffu, hl & 4 ? s[i] : s[i + 4], 4);
      a[i] = __fadd_rn(hl & 4 ? s[i + 4] : s[i], got);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float got = __shfl_xor_sync(0xffffffffu, hl & 2 ? a[i] : a[i + 2], 2);
      b[i] = __fadd_rn(hl & 2 ? a[i + 2] : a[i], got);
    }
    const float got = __shfl_xor_sync(0xffffffffu, hl & 1 ? b[0] : b[1], 1);
    const float c = __fadd_rn(hl & 1 ? b[1] : b[0], got);   // dimension hl of each of the 8 runs of 8
    return shfl_add(shfl_add(shfl_add(c, 4), 2), 1);
  } else {   // unit 4: two runs a lane
    if constexpr (HD == 256) {
#pragma unroll
      for (int i = 0; i < 8; i++) s[i] = shfl_add(s[i], 16);
    }
    const float lo = __fadd_rn(__fadd_rn(__fadd_rn(s[0], s[1]), s[2]), s[3]);
    const float hi = __fadd_rn(__fadd_rn(__fadd_rn(s[4], s[5]), s[6]), s[7]);
    const bool up = threadIdx.x & 8;   // a lane goes on with its first runs, its partner with the second
    const float got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, 8);
    float v = __fadd_rn(up ? hi : lo, got);
    v = shfl_add(shfl_add(shfl_add(v, 4), 2), 1);
    return shfl_add(v, 8);
  }
}

// A warp takes `steps` steps of 32 / (hd / 8) heads of one row: the row's place in
// the cache, its rotation and the norm weights stay in registers.
template <int HD, int BITS, typename In>
__global__ void __launch_bounds__(256, 4) paged_append_kernel(const PagedView c, const AppendParams a) {
  constexpr int L = HD / 8, HPW = 32 / L;   // lanes of a head; heads of a warp's step
  pdl_trigger();
  const int lane = threadIdx.x & 31, hl = lane % L, d0 = hl * 8;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);   // (row, part of its heads)
  if (item >= (int64_t)a.T * a.parts) return;
  const int64_t t = item / a.parts;
  const int n_heads = a.heads + 2 * c.kv_heads, h0 = (int)(item - t * a.parts) * a.steps * HPW;
  pdl_wait();
  const In *src = static_cast<const In *>(a.qkv) + t * a.ld + d0;
  int h = h0 + lane / L;
  Raw<In> next = load_raw(src + (int64_t)min(h, n_heads - 1) * HD);
  const int pos = a.pos[t], seq = a.seq[t];
  const bool fits = a.rot == 0 || (pos >= 0 && pos < a.n_pos);
  const int half = a.rot / 2;
  const bool in = fits && d0 < a.rot, low = d0 < half;
  float cs[8], sn[8], g[8];
  if (in) {
    if (a.pairs) {
      const float4 u = __ldg(reinterpret_cast<const float4 *>(a.cos_t + (int64_t)pos * half + d0 / 2));
      const float4 w = __ldg(reinterpret_cast<const float4 *>(a.sin_t + (int64_t)pos * half + d0 / 2));
      cs[0] = u.x, cs[1] = u.y, cs[2] = u.z, cs[3] = u.w;
      sn[0] = w.x, sn[1] = w.y, sn[2] = w.z, sn[3] = w.w;
    } else {   // x cos + (the other half's) (-sin, sin)
      const int64_t at = (int64_t)pos * half + (low ? d0 : d0 - half);
      load8(a.cos_t + at, cs);
      load8(a.sin_t + at, sn);
#pragma unroll
      for (int i = 0; i < 8; i++) sn[i] = low ? -sn[i] : sn[i];
    }
  }
  uint8_t *blk = paged_block(c, seq, pos);
  const bool ok = blk != nullptr && fits;
  if (!ok && lane == 0) atomicOr(&g_paged_status, SM100_DECODE_ERR_ARG);
  const int row = pos & (c.page - 1);
  const int partner = d0 < a.rot ? (low ? lane + half / 8 : lane - half / 8) : lane;
  // this lane's part of the row's q, and of a key head's keys (values: half a block on)
  __nv_bfloat16 *q_row = a.q_out + t * a.heads * HD + d0;
  uint8_t *kv_row = blk + (BITS == 16 ? ((int64_t)row * HD + d0) * 2 : (int64_t)row * (HD / 2) + hl * 4);
  const int marks = BITS == 16 ? 0 : (c.page - row) * (HD / 2) - hl * 4 + (row * (HD / kGroup) + hl / 8) * 4;
  int kind = -1;   // whose norm weights g holds: 0 queries, 1 keys

  for (int i = 0; i < a.steps && h0 + i * HPW < n_heads; i++, h += HPW) {
    float x[8];
    next.get(x);
    if (h + HPW < n_heads) next = load_raw(src + (int64_t)(h + HPW) * HD);   // the next step's load under way
    const bool live = h < n_heads, is_q = h < a.heads, turns = h < a.heads + c.kv_heads;
    const bool turning = h0 + i * HPW < a.heads + c.kv_heads;   // one of the step's heads is a query or a key
    if (turning && (a.g_q || a.g_k)) {
      const float ss = sum_squares<HD>(x);
      const float *gp = is_q ? a.g_q : a.g_k;
      if (turns && gp) {
        if (kind != !is_q) {
          kind = !is_q;
          load8(gp + d0, g);
        }
        const float r = rsqrtf(__fadd_rn(ss * (1.0f / HD), a.eps));
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __fmul_rn(__fmul_rn(x[j], r), g[j]);
      }
    }
    if (turning && a.rot) {
      if (a.pairs) {
        if (in && turns) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float u = x[2 * j], w = x[2 * j + 1];
            x[2 * j] = __fsub_rn(__fmul_rn(u, cs[j]), __fmul_rn(w, sn[j]));
            x[2 * j + 1] = __fadd_rn(__fmul_rn(w, cs[j]), __fmul_rn(u, sn[j]));
          }
        }
      } else {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = __shfl_sync(0xffffffffu, x[j], partner);
        if (in && turns) {
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = __fadd_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(y[j], sn[j]));
        }
      }
    }
    if (is_q) *reinterpret_cast<uint4 *>(q_row + (int64_t)h * HD) = ok ? pack8(x) : make_uint4(0, 0, 0, 0);
    const bool store = live && ok && !is_q;
    uint8_t *dst = kv_row + (int64_t)(h - a.heads - (turns ? 0 : c.kv_heads)) * c.block + (turns ? 0 : c.block / 2);
    if constexpr (BITS == 16) {
      if (store) *reinterpret_cast<uint4 *>(dst) = pack8(x);
    } else if (h0 + i * HPW + HPW > a.heads) {   // one of the step's heads is kept
      float mn = x[0], mx = x[0];
#pragma unroll
      for (int j = 1; j < 8; j++) mn = min_nan(mn, x[j]), mx = max_nan(mx, x[j]);
#pragma unroll
      for (int o = kGroup / 16; o > 0; o >>= 1) {   // the 8 lanes of a group
        mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      }
      const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(mx, mn), 1.0f / 15.0f)), mb = __float2bfloat16_rn(mn);
      const float s = __bfloat162float(sb), m = __bfloat162float(mb);
      uint32_t codes = 0;
      if (s > 0.0f) {
#pragma unroll
        for (int j = 0; j < 8; j++)
          codes |= (uint32_t)fminf(fmaxf(rintf((x[j] - m) / s), 0.0f), 15.0f) << (4 * j);
      }
      if (store) {
        *reinterpret_cast<uint32_t *>(dst) = codes;
        if (hl % 8 == 0) *reinterpret_cast<__nv_bfloat162 *>(dst + marks) = __halves2bfloat162(sb, mb);
      }
    }
  }
}

template <int HD, int BITS>
__global__ void __launch_bounds__(256) paged_read_kernel(const PagedView c, const int32_t *pos, const int32_t *seq,
                                                         __nv_bfloat16 *k, __nv_bfloat16 *v, int64_t items) {
  constexpr int L = HD / 8;
  pdl_trigger();
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;   // (t, key head, keys | values)
  const int hl = threadIdx.x % L;
  pdl_wait();
  if (item >= items) return;
  const int64_t t = item / (2 * c.kv_heads);
  const int r = (int)(item - t * 2 * c.kv_heads), kh = r >> 1, is_v = r & 1;
  const int p = pos[t];
  const uint8_t *blk = paged_block(c, seq[t], p);
  uint4 out = make_uint4(0, 0, 0, 0);
  if (!blk) {
    if (hl == 0) atomicOr(&g_paged_status, SM100_DECODE_ERR_ARG);
  } else {
    const uint8_t *src = blk + (int64_t)kh * c.block + (is_v ? c.block / 2 : 0);
    const int row = p & (c.page - 1);
    if constexpr (BITS == 16) {
      out = *reinterpret_cast<const uint4 *>(src + ((int64_t)row * HD + hl * 8) * 2);
    } else {
      const uint32_t codes = *reinterpret_cast<const uint32_t *>(src + (int64_t)row * (HD / 2) + hl * 4);
      const uint32_t sm = *reinterpret_cast<const uint32_t *>(src + (int64_t)c.page * (HD / 2) +
                                                              ((int64_t)row * (HD / kGroup) + hl / 8) * 4);
      const float s = bf16_lo(sm), m = bf16_hi(sm);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = __fadd_rn(m, __fmul_rn((float)((codes >> (4 * i)) & 15u), s));
      out = pack8(x);
    }
  }
  *reinterpret_cast<uint4 *>((is_v ? v : k) + (t * c.kv_heads + kh) * HD + hl * 8) = out;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" uint64_t sm100_paged_block_bytes(int32_t page, int32_t head_dim, int32_t bits) {
  if ((page != 16 && page != 32 && page != 64) || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
  if (bits == SM100_KV_BF16) return 4ull * page * head_dim;
  if (bits == SM100_KV_Q4) return 2ull * page * (head_dim / 2 + 4 * (head_dim / kGroup));
  return 0;
}

int sm100_paged_view(const Sm100PagedCache *c, const char *what, PagedView *v) {
  if (!c || !c->pool || !c->table) return sm100_set_error(SM100_ERR_ARG, "%s: no cache", what);
  const uint64_t block = sm100_paged_block_bytes(c->page, c->head_dim, c->bits);
  if (!block)
    return sm100_set_error(SM100_ERR_UNSUPPORTED,
                           "%s: page %d (16, 32, 64), head_dim %d (64, 128, 256), bits %d (4, 16)", what, c->page,
                           c->head_dim, c->bits);
  if (c->n_pages < 1 || c->kv_heads < 1 || c->n_seq < 1 || c->max_pages < 1 ||
      (int64_t)c->max_pages * c->page > 1 << 30 || !aligned16(c->pool))
    return sm100_set_error(SM100_ERR_ARG, "%s: n_pages %d kv_heads %d n_seq %d max_pages %d, pool 16-byte aligned",
                           what, c->n_pages, c->kv_heads, c->n_seq, c->max_pages);
  v->pool = static_cast<uint8_t *>(c->pool);
  v->table = c->table;
  v->n_pages = c->n_pages;
  v->page = c->page;
  v->page_log2 = c->page == 16 ? 4 : c->page == 32 ? 5 : 6;
  v->kv_heads = c->kv_heads;
  v->n_seq = c->n_seq;
  v->max_pages = c->max_pages;
  v->block = (uint32_t)block;
  return SM100_OK;
}

namespace {

template <int HD>
cudaError_t append_hd(const PagedView &v, int bits, int dtype, AppendParams p, cudaStream_t st) {
  // a row's heads in as few warps as still fill the GPU: 16384 rows of 48 heads in bf16 take 92 us with a warp a row, 104
  // with ten steps a warp; 4093 rows of 36 heads in 4 bits (and their reading) 28.8 us with all steps in a warp, 45.9 with one
  const int n_heads = p.heads + 2 * v.kv_heads, hpw = 32 / (HD / 8), all = (n_heads + hpw - 1) / hpw;
  const int64_t even = (int64_t)p.T * all / kAppendWarps;
  p.steps = (int)(even < 1 ? 1 : even < all ? even : all);
  p.parts = (all + p.steps - 1) / p.steps;
  const int64_t blocks = ((int64_t)p.T * p.parts + 7) / 8;
  const dim3 grid((unsigned)blocks), block(256);
  if (bits == 16)
    return dtype == SM100_DT_F32 ? launch_pdl(paged_append_kernel<HD, 16, float>, grid, block, 0, st, v, p)
                                 : launch_pdl(paged_append_kernel<HD, 16, __nv_bfloat16>, grid, block, 0, st, v, p);
  return dtype == SM100_DT_F32 ? launch_pdl(paged_append_kernel<HD, 4, float>, grid, block, 0, st, v, p)
                               : launch_pdl(paged_append_kernel<HD, 4, __nv_bfloat16>, grid, block, 0, st, v, p);
}

}  // namespace

extern "C" int sm100_paged_append(const Sm100PagedCache *c, const Sm100PagedAppendArgs *a, void *stream) {
  PagedView v;
  if (int rc = sm100_paged_view(c, "paged_append", &v)) return rc;
  if (a && a->T == 0) return SM100_OK;
  if (!a || !a->qkv || !a->pos || !a->seq || !a->q_out || a->T < 0 || a->heads < 1 || a->heads % c->kv_heads)
    return sm100_set_error(SM100_ERR_ARG, "paged_append: T %d heads %d (a multiple of kv_heads %d)", a ? a->T : 0,
                           a ? a->heads : 0, c->kv_heads);
  if (a->dtype != SM100_DT_F32 && a->dtype != SM100_DT_BF16)
    return sm100_set_error(SM100_ERR_UNSUPPORTED, "paged_append: qkv dtype %d (f32 or bf16)", a->dtype);
  const int64_t n_heads = (int64_t)a->heads + 2 * (int64_t)c->kv_heads;
  if (a->T * n_heads >= INT32_MAX)
    return sm100_set_error(SM100_ERR_ARG, "paged_append: %d rows of %lld heads in one call", a->T, (long long)n_heads);
  const int64_t width = n_heads * c->head_dim, ld = a->ld ? a->ld : width;
  const bool rot = a->cos_t || a->sin_t;
  if (rot && (!a->cos_t || !a->sin_t || a->rot < 16 || a->rot % 16 || a->rot > c->head_dim || a->n_pos < 1 ||
              !aligned16(a->cos_t) || !aligned16(a->sin_t)))
    return sm100_set_error(SM100_ERR_ARG, "paged_append: rot %d (a multiple of 16 up to head_dim), n_pos %d, both tables",
                           a->rot, a->n_pos);
  if (ld < width || ld % (a->dtype == SM100_DT_F32 ? 4 : 8) || !aligned16(a->qkv) || !aligned16(a->q_out) ||
      (a->g_q && !aligned16(a->g_q)) || (a->g_k && !aligned16(a->g_k)))
    return sm100_set_error(SM100_ERR_ARG, "paged_append: row stride %lld of %lld elements, 16-byte rows and addresses",
                           (long long)ld, (long long)width);
  AppendParams p{a->qkv, a->g_q, a->g_k, a->cos_t, a->sin_t, a->pos, a->seq, static_cast<__nv_bfloat16 *>(a->q_out),
                 ld, a->T, a->heads, rot ? a->rot : 0, a->n_pos, a->pairs, 0, 0, a->eps};
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = c->head_dim == 64    ? append_hd<64>(v, c->bits, a->dtype, p, st)
                        : c->head_dim == 128 ? append_hd<128>(v, c->bits, a->dtype, p, st)
                                             : append_hd<256>(v, c->bits, a->dtype, p, st);
  if (e != cudaSuccess) return sm100_set_error(SM100_ERR_CUDA, "paged_append: %s", cudaGetErrorString(e));
  return launch_status("paged_append");
}

extern "C" int sm100_paged_read(const Sm100PagedCache *c, const int32_t *pos, const int32_t *seq, void *k, void *v,
                                int32_t T, void *stream) {
  PagedView w;
  if (int rc = sm100_paged_view(c, "paged_read", &w)) return rc;
  if (T == 0) return SM100_OK;
  if (!pos || !seq || !k || !v || T < 0 || !aligned16(k) || !aligned16(v))
    return sm100_set_error(SM100_ERR_ARG, "paged_read: T %d, k and v 16-byte aligned", T);
  const int64_t items = (int64_t)T * 2 * c->kv_heads, blocks = (items * (c->head_dim / 8) + 255) / 256;
  if (blocks >= INT32_MAX) return sm100_set_error(SM100_ERR_ARG, "paged_read: %d rows in one call", T);
  const dim3 grid((unsigned)blocks), block(256);
  auto *ko = static_cast<__nv_bfloat16 *>(k), *vo = static_cast<__nv_bfloat16 *>(v);
  cudaStream_t st = (cudaStream_t)stream;
  const bool q4 = c->bits == SM100_KV_Q4;
  cudaError_t e;
  if (c->head_dim == 64)
    e = q4 ? launch_pdl(paged_read_kernel<64, 4>, grid, block, 0, st, w, pos, seq, ko, vo, items)
           : launch_pdl(paged_read_kernel<64, 16>, grid, block, 0, st, w, pos, seq, ko, vo, items);
  else if (c->head_dim == 128)
    e = q4 ? launch_pdl(paged_read_kernel<128, 4>, grid, block, 0, st, w, pos, seq, ko, vo, items)
           : launch_pdl(paged_read_kernel<128, 16>, grid, block, 0, st, w, pos, seq, ko, vo, items);
  else
    e = q4 ? launch_pdl(paged_read_kernel<256, 4>, grid, block, 0, st, w, pos, seq, ko, vo, items)
           : launch_pdl(paged_read_kernel<256, 16>, grid, block, 0, st, w, pos, seq, ko, vo, items);
  if (e != cudaSuccess) return sm100_set_error(SM100_ERR_CUDA, "paged_read: %s", cudaGetErrorString(e));
  return launch_status("paged_read");
}

extern "C" uint32_t sm100_paged_status(void) {
  uint32_t v = 0, z = 0;
  cudaDeviceSynchronize();
  cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(v));
  cudaMemcpyToSymbol(g_paged_status, &z, sizeof(z));
  return v | sm100_paged_attn_take_status();
}
