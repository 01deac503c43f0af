// The next ids from logits: temperature, top-k, top-p and min-p, then a race
// on given exponential random numbers.
//
// With ids in the order of falling logit (equal ones by rising id) every filter
// keeps a beginning of the order, so what is kept is one cut: the ids at or
// before a place in the order.  A place is a 64-bit key, the logit's bits made
// monotonic above the complement of the id, and larger keys come first.
//   top-k: the largest key with at least k keys at or above it
//   top-p: the smallest key whose forerunners weigh less than p * (weight of
//          what top-k left)
//   min-p: w >= min_p, monotonic in the logit
// The kept id with the largest d - ln(noise) wins: -ln of an exponential number
// is a Gumbel number, so id i wins with probability w_i / sum w.
//
// One CTA per row; each cut is a bisection over the 64 bits of the key.
#include "common.cuh"

#include <float.h>

using namespace sm100;

namespace {

constexpr int kThreads = 512;

struct SampleParams {
  const void *logits;
  const float *noise, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  int32_t *tok;
  float *logp;
  int64_t ld, ld_noise;
  int V;
};

__device__ __forceinline__ float logit_at(const float *p, int64_t i) { return p[i]; }
__device__ __forceinline__ float logit_at(const __nv_bfloat16 *p, int64_t i) { return __bfloat162float(p[i]); }

__device__ __forceinline__ uint64_t place(float l, int i) {   // 0: left out
  if (!(l > -INFINITY)) return 0;
  l = fminf(l, FLT_MAX) + 0.0f;   // -0 and 0 are equal logits
  const uint32_t u = __float_as_uint(l);
  const uint32_t key = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)key << 32 | (uint32_t)~i;
}

__device__ __forceinline__ float logit_of(uint64_t pl) {
  const uint32_t key = (uint32_t)(pl >> 32);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ uint64_t block_max64(uint64_t v, uint64_t *red) {
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int i = 0; i < kThreads / 32; i++) v = red[i] > v ? red[i] : v;
  return v;
}

__device__ uint64_t block_sum64(uint64_t v, uint64_t *red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kThreads / 32; i++) v += red[i];
  return v;
}

// A weight e^d <= 1 in units of 2^-40: sums of them are exact in 64 bits (V <
// 2^23), so a cut by weight depends on no order of summation.
__device__ __forceinline__ uint64_t fixed(float w) { return __float2ull_rn(w * 1099511627776.0f); }

template <typename In>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams a) {
  __shared__ uint64_t red[kThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, tid = threadIdx.x;
  const In *row = static_cast<const In *>(a.logits) + b * a.ld;
  uint64_t top = 0;
  for (int i = tid; i < a.V; i += kThreads) {
    const uint64_t pl = place(logit_at(row, i), i);
    top = pl > top ? pl : top;
  }
  top = block_max64(top, red);
  const float T = a.temperature ? a.temperature[b] : 1.0f;
  if (top == 0 || !(T > 0.0f)) {
    if (tid == 0) {
      a.tok[b] = top == 0 ? -1 : (int32_t)~(uint32_t)top;
      if (a.logp) a.logp[b] = top == 0 ? -INFINITY : 0.0f;
    }
    return;
  }
  const float lmax = logit_of(top);
  uint64_t cut = 1;   // kept: place >= cut
  const int k = a.top_k ? a.top_k[b] : 0;
  if (k > 0 && k < a.V) {
    uint64_t lo = 0;   // the largest place with at least k places at or above it (0 where there are fewer)
    for (int bit = 63; bit >= 0; bit--) {
      const uint64_t mid = lo | 1ull << bit;
      uint64_t n = 0;
      for (int i = tid; i < a.V; i += kThreads) n += place(logit_at(row, i), i) >= mid;
      if (block_sum64(n, red) >= (uint64_t)k) lo = mid;
    }
    cut = lo ? lo : 1;
  }
  const float p = a.top_p ? a.top_p[b] : 1.0f;
  if (p < 1.0f) {
    uint64_t all = 0;
    for (int i = tid; i < a.V; i += kThreads) {
      const uint64_t pl = place(logit_at(row, i), i);
      if (pl >= cut) all += fixed(expf((logit_of(pl) - lmax) / T));
    }
    const double target = (double)p * (double)block_sum64(all, red);
    uint64_t lo = 0;   // the largest number with at least the target's weight above it: the cut is the next
    for (int bit = 63; bit >= 0; bit--) {
      const uint64_t mid = lo | 1ull << bit;
      uint64_t m = 0;
      for (int i = tid; i < a.V; i += kThreads) {
        const uint64_t pl = place(logit_at(row, i), i);
        if (pl > mid && pl >= cut) m += fixed(expf((logit_of(pl) - lmax) / T));
      }
      if ((double)block_sum64(m, red) >= target) lo = mid;
    }
    cut = lo >= top ? top : lo + 1 > cut ? lo + 1 : cut;
  }
  const float min_p = a.min_p ? a.min_p[b] : 0.0f;
  const float *noise = a.noise + b * a.ld_noise;
  uint64_t kept = 0;
  float best = -INFINITY;
  int best_i = -1;
  for (int i = tid; i < a.V; i += kThreads) {
    const uint64_t pl = place(logit_at(row, i), i);
    if (pl < cut) continue;
    const float d = (logit_of(pl) - lmax) / T, w = expf(d);
    if (!(w >= min_p) && pl != top) continue;
    kept += fixed(w);
    const float s = d - logf(noise[i]);
    if (s > best) best = s, best_i = i;   // i rises: equal scores keep the lower id
  }
  kept = block_sum64(kept, red);
  const uint64_t mine = best_i < 0 ? 0 : place(best, best_i);   // place() clamps +inf; -inf never became best
  const uint64_t won = block_max64(mine, red);
  if (tid == 0) {
    const int id = (int32_t)~(uint32_t)(won ? won : top);
    a.tok[b] = id;
    if (a.logp) a.logp[b] = (logit_of(place(logit_at(row, id), id)) - lmax) / T - logf((float)kept * 0x1p-40f);
  }
}

}  // namespace

extern "C" int sm100_sample(const Sm100SampleArgs *a, void *stream) {
  if (a && a->B == 0) return SM100_OK;
  if (!a || !a->logits || !a->noise || !a->tok || a->B < 0 || a->V < 1 || a->V >= 1 << 23 || a->ld < 0 || a->ld_noise < 0 ||
      (a->ld && a->ld < a->V) || (a->ld_noise && a->ld_noise < a->V))
    return sm100_set_error(SM100_ERR_ARG, "sample: B %d V %d (1 .. 2^23 - 1) ld %lld ld_noise %lld", a ? a->B : 0, a ? a->V : 0,
                           a ? (long long)a->ld : 0, a ? (long long)a->ld_noise : 0);
  if (a->dtype != SM100_DT_F32 && a->dtype != SM100_DT_BF16)
    return sm100_set_error(SM100_ERR_UNSUPPORTED, "sample: logits dtype %d (f32 or bf16)", a->dtype);
  const SampleParams p{a->logits, a->noise, a->temperature, a->top_k, a->top_p, a->min_p, a->tok, a->logp,
                       a->ld ? a->ld : a->V, a->ld_noise ? a->ld_noise : a->V, a->V};
  const cudaError_t e =
      a->dtype == SM100_DT_F32
          ? launch_pdl(sample_kernel<float>, dim3(a->B), dim3(kThreads), 0, (cudaStream_t)stream, p)
          : launch_pdl(sample_kernel<__nv_bfloat16>, dim3(a->B), dim3(kThreads), 0, (cudaStream_t)stream, p);
  if (e != cudaSuccess) return sm100_set_error(SM100_ERR_CUDA, "sample: %s", cudaGetErrorString(e));
  return launch_status("sample");
}
