// Attention of new rows over the paged key / value cache: out = softmax(q k^T
// scale) v, query head h on key head h / (heads / kv_heads), row r of n on keys
// 0 .. kv_len - n + r.
//
// One CTA per (row, query head): each of four warps takes every fourth key,
// its lanes the dimensions, with a running maximum and sum; the warps' parts
// are joined in shared memory.
#include "paged.cuh"

using namespace sm100;

namespace {

struct AttnParams {
  const __nv_bfloat16 *q;
  const int32_t *kv_len, *q_off;
  __nv_bfloat16 *out;
  int64_t ld_q;
  int T, heads, max_rows;
  float scale;
};

template <int HD, int BITS>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedView c, const AttnParams a) {
  constexpr int E = HD / 32;   // dimensions of a lane: lane * E ..
  __shared__ float part[4][HD + 2];
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x / a.heads, h = blockIdx.x % a.heads, kh = h / (a.heads / c.kv_heads);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = t, first = t, n = 1;
  if (a.q_off) {   // the sequence whose rows hold row t
    int lo = 0, hi = c.n_seq - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (a.q_off[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    s = lo, first = a.q_off[s], n = a.q_off[s + 1] - first;
  }
  int len = a.kv_len[s];
  if (len > c.max_pages * c.page) {
    len = c.max_pages * c.page;
    if (threadIdx.x == 0) atomicOr(&g_paged_status, SM100_DECODE_ERR_ARG);
  }
  const int keys = len - n + (t - first) + 1;
  float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < E; i++) q[i] = __bfloat162float(a.q[t * a.ld_q + (int64_t)h * HD + lane * E + i]) * a.scale;
  for (int j = warp; j < keys; j += 4) {
    const uint8_t *blk = paged_block(c, s, j);
    if (!blk) {
      if (lane == 0) atomicOr(&g_paged_status, SM100_DECODE_ERR_ARG);
      continue;
    }
    const int row = j & (c.page - 1);
    float k[E], v[E];
#pragma unroll
    for (int w = 0; w < 2; w++) {
      const uint8_t *src = blk + (int64_t)kh * c.block + w * (c.block / 2);
      float *x = w ? v : k;
#pragma unroll
      for (int i = 0; i < E; i++) {
        const int d = lane * E + i;
        if constexpr (BITS == 16) {
          x[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(src)[row * HD + d]);
        } else {
          const __nv_bfloat162 sm = *reinterpret_cast<const __nv_bfloat162 *>(src + c.page * (HD / 2) +
                                                                              (row * (HD / kGroup) + d / kGroup) * 4);
          const uint32_t code = (src[row * (HD / 2) + d / 2] >> (4 * (d & 1))) & 15u;
          x[i] = __high2float(sm) + (float)code * __low2float(sm);
        }
      }
    }
    float z = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) z = fmaf(q[i], k[i], z);
    z = warp_sum(z);
    const float mn = fmaxf(m, z), f = __expf(m - mn), p = __expf(z - mn);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < E; i++) o[i] = o[i] * f + p * v[i];
    m = mn;
  }
#pragma unroll
  for (int i = 0; i < E; i++) part[warp][lane * E + i] = o[i];
  if (lane == 0) part[warp][HD] = m, part[warp][HD + 1] = l;
  __syncthreads();
  float mx = -INFINITY;
  for (int w = 0; w < 4; w++) mx = fmaxf(mx, part[w][HD]);
  for (int d = threadIdx.x; d < HD; d += 128) {
    float num = 0.0f, den = 0.0f;
    for (int w = 0; w < 4; w++) {
      if (part[w][HD + 1] == 0.0f) continue;
      const float f = __expf(part[w][HD] - mx);
      num += part[w][d] * f;
      den += part[w][HD + 1] * f;
    }
    a.out[((int64_t)t * a.heads + h) * HD + d] = __float2bfloat16_rn(keys > 0 && den != 0.0f ? num / den : 0.0f);
  }
}

template <int HD>
cudaError_t attn_hd(const PagedView &v, int bits, const AttnParams &p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.T * p.heads)), block(128);
  return bits == 4 ? launch_pdl(paged_attn_kernel<HD, 4>, grid, block, 0, st, v, p)
                   : launch_pdl(paged_attn_kernel<HD, 16>, grid, block, 0, st, v, p);
}

}  // namespace

extern "C" uint64_t sm100_paged_attention_ws_bytes(const Sm100PagedCache *c, int32_t heads, int32_t max_rows) {
  PagedView v;
  if (sm100_paged_view(c, "paged_attention_ws_bytes", &v) || heads < 1 || heads % c->kv_heads || max_rows < 1) return 0;
  return 16;
}

extern "C" int sm100_paged_attention(const Sm100PagedCache *c, const Sm100PagedAttnArgs *a, void *stream) {
  PagedView v;
  if (int rc = sm100_paged_view(c, "paged_attention", &v)) return rc;
  if (a && a->T == 0) return SM100_OK;
  if (!a || !a->q || !a->kv_len || !a->out || !a->ws || a->T < 0 || a->heads < 1 || a->heads % c->kv_heads ||
      a->max_rows < 1 || (!a->q_off && (a->T != c->n_seq || a->max_rows != 1)))
    return sm100_set_error(SM100_ERR_ARG,
                           "paged_attention: T %d (n_seq %d without q_off) heads %d (a multiple of kv_heads %d) "
                           "max_rows %d", a ? a->T : 0, c->n_seq, a ? a->heads : 0, c->kv_heads, a ? a->max_rows : 0);
  const int64_t width = (int64_t)a->heads * c->head_dim, ld = a->ld_q ? a->ld_q : width;
  if (ld < width || ld % 8 || ((uintptr_t)a->q & 15) || ((uintptr_t)a->out & 15) || ((uintptr_t)a->ws & 15))
    return sm100_set_error(SM100_ERR_ARG, "paged_attention: q stride %lld of %lld, 16-byte rows and addresses",
                           (long long)ld, (long long)width);
  const uint64_t need = sm100_paged_attention_ws_bytes(c, a->heads, a->max_rows);
  if (a->ws_bytes < need)
    return sm100_set_error(SM100_ERR_ARG, "paged_attention: %llu bytes of scratch, %llu needed",
                           (unsigned long long)a->ws_bytes, (unsigned long long)need);
  const AttnParams p{static_cast<const __nv_bfloat16 *>(a->q), a->kv_len, a->q_off,
                     static_cast<__nv_bfloat16 *>(a->out), ld, a->T, a->heads, a->max_rows, a->scale};
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = c->head_dim == 64    ? attn_hd<64>(v, c->bits, p, st)
                        : c->head_dim == 128 ? attn_hd<128>(v, c->bits, p, st)
                                             : attn_hd<256>(v, c->bits, p, st);
  if (e != cudaSuccess) return sm100_set_error(SM100_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
  return launch_status("paged_attention");
}

uint32_t sm100_paged_attn_take_status(void) {
  uint32_t v = 0, z = 0;
  cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(v));
  cudaMemcpyToSymbol(g_paged_status, &z, sizeof(z));
  return v;
}
