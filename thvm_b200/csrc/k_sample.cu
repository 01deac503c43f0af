// The next ids from logits: temperature, top-k, top-p and min-p, then a race
// on given exponential random numbers.
//
// With ids in the order of falling logit (equal ones by rising id) every filter
// keeps a beginning of the order, so what is kept is one cut, a place in the
// order.  A place is a 64-bit key, the logit's bits made monotonic above the
// complement of the id; larger keys come first.
//   top-k: the last place with fewer than k places before it
//   top-p: the last place whose forerunners weigh less than p * (weight of what
//          top-k left)
//   min-p: w >= min_p, monotonic in the logit
// The kept id with the largest d - ln(noise) wins: -ln of an exponential number
// is a Gumbel number, so id i wins with probability w_i / sum w.
//
// What bounds it: the logits once, and the random numbers of the kept ids.  A
// row belongs to a cluster of 1 to 8 CTAs, as many as hold it in their shared
// memory (and as fill the GPU where there are few rows), so every later pass is
// over shared memory.  A cut is found without sorting the row:
//   1. a histogram of (l_max - l) / T in 4096 bins of 1/128, summed over the
//      cluster slice by slice;
//   2. the bins that can hold the cut: by count it is one; by weight a bin's
//      ids weigh count * e^-bin within e^(+-1/256), which bounds the cut to some
//      bins, and where those hold too many ids, narrower bounds about a guess
//      that knows the row's whole weight;
//   3. one pass sums what lies above those bins and gathers their ids (a few
//      hundred), which CTA 0 sorts and scans; a guess that missed is put right
//      by what the pass summed.
// Where everything above the cut fits in the list too (top-k of up to some
// hundreds, a peaked top-p) the list is all that is kept, and CTA 0 runs the
// race on it alone.  A bin that overflows the list (thousands of equal logits at
// the cut) falls back to a bisection over the 64 bits of a place.
// A thread sums the weights of its few dozen ids in f32, in a fixed order; from
// there on sums are 64-bit integers in units of 2^-40, so no order of arrival
// enters a result.
#include "common.cuh"

#include <cooperative_groups.h>
#include <float.h>

namespace cg = cooperative_groups;
using namespace sm100;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 4096, kCap = 2048, kMaxCtas = 8;
constexpr float kPerNat = 128.0f;

struct SampleParams {
  const void *logits;
  const float *noise, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  int32_t *tok;
  float *logp;
  int64_t ld, ld_noise;
  int V, chunk;            // chunk: ids of a CTA, a multiple of 16
  int vec, noise_vec;      // rows on 16 bytes
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float &o) { o = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }

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

__device__ __forceinline__ int id_of(uint64_t pl) { return (int)~(uint32_t)pl; }

// A weight, or a thread's sum of some, in units of 2^-40
__device__ __forceinline__ uint64_t fixed(float w) { return __float2ull_rn(w * 1099511627776.0f); }

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// A row's logits as weights: w = e^((l - l_max) / T) = 2^(x c), c = log2(e) / T
// in two floats, the product's rounding carried along: ~2^-22 of w at any
// distance, without a division per id.
struct Scale {
  float lmax, T, hi, lo, per;
  __device__ void set(float top, float t) {
    lmax = top, T = t;
    const double c = fmin(1.4426950408889634 / (double)t, 1e38);
    hi = (float)c;
    lo = (float)(c - (double)hi);
    per = fminf(kPerNat / t, 1e38f);
  }
  __device__ __forceinline__ float below(float l) const { return fminf(l, FLT_MAX) - lmax; }
  __device__ __forceinline__ float weight(float l) const {
    const float x = below(l), t = x * hi;
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(t));
    const float e = fmaf(x, lo, fmaf(x, hi, -t));
    return t < -125.0f ? 0.0f : fmaf(w * e, 0.6931472f, w);
  }
  // bins of 1 / kPerNat around their multiples; the last takes everything further off
  __device__ __forceinline__ int bin(float l) const {
    const float v = fminf(-below(l) * per, (float)(kBins - 1));
    return __float_as_int(v + 12582912.0f) & 0x3fffff;   // to the nearest integer
  }
  __device__ __forceinline__ float d(float l) const { return below(l) / T; }
};

// A sum reaches `goal` in bin `bin`; ids and estimated weight before the bin,
// ids up to its end.
struct Crossing {
  int bin;
  uint32_t before, upto;
  float weight_before;
};

enum { kSureLo, kSureHi, kWideLo, kWideHi, kNearLo, kNearHi, kGuess, kGoals };

struct alignas(16) Shared {
  uint64_t list[kCap];
  uint32_t hist[kBins];
  uint64_t red[kWarps], red2[kWarps];
  // read by the other CTAs of the cluster
  uint64_t top, row, above, best, kept;   // largest place; weight of all ids; measure above the bins; winner; kept weight
  uint32_t n_list, ids;                   // gathered places; ids in this CTA's slice of bins
  float heavy;                            // and their estimated weight
  // of CTA 0, written by whoever finds it
  Crossing cross[kGoals];
  uint64_t cut, sum, over;
  uint32_t done, missed;
};

__device__ __forceinline__ uint64_t block_sum64(uint64_t v, uint64_t *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (kWarps - 1)];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ uint64_t block_max64(uint64_t v, uint64_t *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max64(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (kWarps - 1)];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) v = max64(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Sum of the values of the threads before this one; total in *all.
template <typename T>
__device__ __forceinline__ T block_before(T v, T *red, T *all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T up = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T x = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += x;
  }
  __syncthreads();
  if (lane == 31) red[warp] = up;
  __syncthreads();
  T w = lane < kWarps ? red[lane] : T(0);
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const T x = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += x;
  }
  *all = __shfl_sync(0xffffffffu, w, kWarps - 1);
  const T before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return (warp ? before : T(0)) + up - v;
}

template <typename In, bool RESIDENT>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams a) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shared sh;
  constexpr int E = 16 / sizeof(In);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x;
  const int b = blockIdx.x / C;
  pdl_trigger();
  for (int i = tid; i < kBins; i += kThreads) sh.hist[i] = 0;
  pdl_wait();
  const int begin = min(rank * a.chunk, a.V), n = min(a.V - begin, a.chunk);
  const In *src = static_cast<const In *>(a.logits) + b * a.ld + begin;
  In *held = reinterpret_cast<In *>(dyn);
  // every id of the CTA (l, i), a thread's in rising order; in shared memory 16 bytes at a time, the end filled up with -inf
  const int nv = (n + E - 1) / E;
  const auto each = [&](auto f) {
    if constexpr (RESIDENT) {
      for (int i = tid; i < nv; i += kThreads) {
        const uint4 v = reinterpret_cast<const uint4 *>(held)[i];
        const In *x = reinterpret_cast<const In *>(&v);
#pragma unroll
        for (int e = 0; e < E; e++) f(to_float(x[e]), i * E + e);
      }
    } else {
#pragma unroll 4
      for (int i = tid; i < n; i += kThreads) f(to_float(__ldg(src + i)), i);
    }
  };
  const float T = a.temperature ? a.temperature[b] : 1.0f;

  // ---- the row into shared memory, and its first place
  float lmax = -INFINITY;
  int imax = 0;
  const auto see = [&](float l, int i) {   // i rises: equal logits keep the lower id
    if (l > lmax) lmax = l, imax = i;
  };
  if (RESIDENT && a.vec) {
    const int whole = n / E;
#pragma unroll 4
    for (int i = tid; i < whole; i += kThreads) {
      const uint4 v = ld_stream_u4(src + (int64_t)i * E);
      reinterpret_cast<uint4 *>(held)[i] = v;
      const In *x = reinterpret_cast<const In *>(&v);
#pragma unroll
      for (int e = 0; e < E; e++) see(to_float(x[e]), i * E + e);
    }
    const int i = whole * E + tid;
    if (tid < nv * E - whole * E) {
      In v;
      from_float(-INFINITY, v);
      if (i < n) v = __ldg(src + i);
      held[i] = v;
      see(to_float(v), i);
    }
  } else {
    const int end = RESIDENT ? nv * E : n;
#pragma unroll 8
    for (int i = tid; i < end; i += kThreads) {
      In v;
      from_float(-INFINITY, v);
      if (i < n) v = __ldg(src + i);
      if (RESIDENT) held[i] = v;
      see(to_float(v), i);
    }
  }
  uint64_t top = block_max64(lmax > -INFINITY ? place(lmax, begin + imax) : 0, sh.red);
  if (tid == 0) sh.top = top, sh.n_list = 0;
  cluster.sync();
  // a value of every CTA of the cluster by the lanes of each warp: one round trip
  const Shared *peer = cluster.map_shared_rank(&sh, (tid & 31) % C);
  const auto cluster_sum = [&](uint64_t v) {
    v = (tid & 31) < C ? v : 0;
#pragma unroll
    for (int o = kMaxCtas / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
  };
  const auto cluster_max = [&](uint64_t v) {
    v = (tid & 31) < C ? v : 0;
#pragma unroll
    for (int o = kMaxCtas / 2; o > 0; o >>= 1) v = max64(v, __shfl_xor_sync(0xffffffffu, v, o));
    return __shfl_sync(0xffffffffu, v, 0);
  };
  top = cluster_max(peer->top);
  if (top == 0 || !(T > 0.0f)) {
    if (rank == 0 && tid == 0) {
      a.tok[b] = top == 0 ? -1 : id_of(top);
      if (a.logp) a.logp[b] = top == 0 ? -INFINITY : 0.0f;
    }
    cluster.sync();   // the others may still read this CTA's first place
    return;
  }
  Scale sc;
  sc.set(logit_of(top), T);
  const float min_p = a.min_p ? a.min_p[b] : 0.0f, p = a.top_p ? a.top_p[b] : 1.0f;
  const int k = a.top_k ? a.top_k[b] : 0;
  Shared *first = cluster.map_shared_rank(&sh, 0);
  // the weight of the cluster's ids that pass a test
  const auto weigh_all = [&](auto test) {
    float w = 0.0f;
    each([&](float l, int i) {
      if (l > -INFINITY && test(l, i)) w += sc.weight(l);
    });
    const uint64_t s = block_sum64(fixed(w), sh.red);
    if (tid == 0) sh.row = s;
    cluster.sync();
    const uint64_t all = cluster_sum(peer->row);
    cluster.sync();
    return all;
  };

  uint64_t cut = 1;   // kept: place >= cut
  bool by_count = k > 0 && k < a.V;
  const bool by_weight = p < 1.0f;
  if (by_count || by_weight) {
    // ---- the histogram, and the weight of the row
    float w = 0.0f;
    each([&](float l, int i) {
      if (!(l > -INFINITY)) return;
      atomicAdd(&sh.hist[sc.bin(l)], 1u);
      if (by_weight) w += sc.weight(l);
    });
    if (by_weight) {
      const uint64_t s = block_sum64(fixed(w), sh.red);
      if (tid == 0) sh.row = s;
    }
    cluster.sync();
    // a CTA sums a slice of the bins over the cluster: kB neighbouring bins a thread
    const int slice = kBins / C, kB = max(slice / kThreads, 1), bin0 = rank * slice + tid * kB;
    const bool mine = tid * kB < slice;
    uint32_t cnt[kBins / kThreads];
#pragma unroll
    for (int i = 0; i < kBins / kThreads; i++) cnt[i] = 0;
    if (mine) {
#pragma unroll
      for (int r = 0; r < kMaxCtas; r++) {
        if (r >= C) break;
        const uint32_t *h = cluster.map_shared_rank(&sh, r)->hist + bin0;
#pragma unroll
        for (int i = 0; i < kBins / kThreads; i++)
          if (i < kB) cnt[i] += h[i];
      }
    }
    uint64_t total = by_weight ? cluster_sum(peer->row) : 0;   // what a top-p is a part of
    uint32_t ids = 0, c_before;
    float heavy = 0.0f, w_before;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; i++)
      if (i < kB) ids += cnt[i], heavy += cnt[i] * __expf(-(float)(bin0 + i) / kPerNat);
    c_before = block_before(ids, reinterpret_cast<uint32_t *>(sh.red), &ids);
    w_before = block_before(heavy, reinterpret_cast<float *>(sh.red2), &heavy);
    if (tid == 0) sh.ids = ids, sh.heavy = heavy;
    cluster.sync();
    uint32_t valid = 0;
    float heavy_all = 0.0f;
    {
      const uint32_t c = (tid & 31) < C ? peer->ids : 0;
      const float h = (tid & 31) < C ? peer->heavy : 0.0f;
#pragma unroll
      for (int r = 0; r < kMaxCtas; r++) {
        const uint32_t cr = __shfl_sync(0xffffffffu, c, r);
        const float hr = __shfl_sync(0xffffffffu, h, r);
        if (r < rank) c_before += cr, w_before += hr;
        valid += cr, heavy_all += hr;
      }
    }
    if (by_count && (uint32_t)k >= valid) by_count = false;   // top-k leaves every id there is

    int last_bin = kBins - 1;   // bins past it are cut off already
    for (int round = by_count ? 0 : 1; round < (by_weight ? 2 : 1); round++) {
      const bool weigh = round == 1;
      // the cut: the last place whose forerunners measure less than target
      const double target = weigh ? (double)p * (double)total : (double)k;
      const float goal = fmaxf((float)(target * (weigh ? 0x1p-40 : 1.0)), 1e-30f);
      // by weight a bin's estimate is within e^(1/256) of its weight.  The guess takes the row's whole weight as known and
      // estimates what lies past the cut: what is off there is the average of many light ids, not a few heavy ones
      float guess = weigh && last_bin == kBins - 1 ? goal - ((float)total * 0x1p-40f - heavy_all) : goal;
      bool bisect = true;
      for (int attempt = 0; attempt < 4; attempt++) {
        if (rank == 0 && tid < kGoals) sh.cross[tid] = Crossing{last_bin, 0, valid, 0.0f};
        if (rank == 0 && tid == 0) sh.done = 0, sh.missed = 0;
        cluster.sync();
        if (mine) {
          const float spread = weigh ? 1.0f : 0.0f;
          const float goals[kGoals] = {goal * (1.0f - 0.0045f * spread), goal * (1.0f + 0.0045f * spread),
                                       guess * (1.0f - 0.001f * spread), guess * (1.0f + 0.001f * spread),
                                       guess * (1.0f - 0.0002f * spread), guess * (1.0f + 0.0002f * spread), guess};
          uint32_t cc = c_before;
          float ww = w_before;
#pragma unroll
          for (int i = 0; i < kBins / kThreads; i++) {
            if (i >= kB || cnt[i] == 0 || bin0 + i > last_bin) continue;
            const uint32_t c1 = cc + cnt[i];
            const float w1 = ww + cnt[i] * __expf(-(float)(bin0 + i) / kPerNat);
#pragma unroll
            for (int g = 0; g < kGoals; g++) {
              const float was = weigh ? ww : (float)cc, now = weigh ? w1 : (float)c1;
              if (now >= goals[g] && (was < goals[g] || cc == 0)) first->cross[g] = Crossing{bin0 + i, cc, c1, ww};
            }
            cc = c1, ww = w1;
          }
        }
        cluster.sync();
        // the widest bounds whose ids fit in the list; from the first id on, where those do
        int lo = 0, hi = 0;
        float before = 0.0f;
        bool fits = false;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const Crossing x = first->cross[g < 3 ? 2 * g : kGuess], y = first->cross[g < 3 ? 2 * g + 1 : kGuess];
          if (g == 0 && attempt) continue;   // the guess knows more by now
          if (fits) continue;
          if (y.upto <= kCap) fits = true, lo = 0, before = 0.0f, hi = y.bin;
          else if (y.upto - x.before <= kCap) fits = true, lo = x.bin, before = x.weight_before, hi = y.bin;
        }
        if (!fits) break;
        float over = 0.0f;
        uint32_t n_over = 0;
        each([&](float l, int i) {
          if (!(l > -INFINITY)) return;
          const int bin = sc.bin(l);
          if (bin > hi) return;
          if (bin < lo) {
            if (weigh) over += sc.weight(l);
            else n_over++;
            return;
          }
          const uint64_t pl = place(l, begin + i);
          if (pl < cut) return;
          const uint32_t x = atomicAdd(&sh.n_list, 1u);
          if (x < kCap) sh.list[x] = pl;
        });
        if (lo > 0) {
          const uint64_t s = block_sum64(weigh ? fixed(over) : n_over, sh.red);
          if (tid == 0) sh.above = s;
        } else if (tid == 0) {
          sh.above = 0;
        }
        cluster.sync();
        if (rank == 0) {
          // the other CTAs' places behind this one's
          const uint32_t c = (tid & 31) < C ? min(peer->n_list, (uint32_t)kCap) : 0;
          const uint64_t above = cluster_sum(peer->above);
          uint32_t m = __shfl_sync(0xffffffffu, c, 0);
#pragma unroll
          for (int r = 1; r < kMaxCtas; r++) {
            const uint32_t cr = min(__shfl_sync(0xffffffffu, c, r), kCap - m);
            if (r < C)
              for (uint32_t i = tid; i < cr; i += kThreads) sh.list[m + i] = cluster.map_shared_rank(&sh, r)->list[i];
            m += cr;
          }
          uint32_t pow2 = 32;
          while (pow2 < m) pow2 *= 2;
          for (uint32_t i = m + tid; i < pow2; i += kThreads) sh.list[i] = 0;
          __syncthreads();
          for (uint32_t size = 2; size <= pow2; size *= 2)   // falling order
            for (uint32_t step = size / 2; step > 0; step /= 2) {
              for (uint32_t i = tid; i < pow2 / 2; i += kThreads) {
                const uint32_t x = 2 * i - (i & (step - 1)), y = x + step;
                const uint64_t u = sh.list[x], v = sh.list[y];
                if ((u < v) == !(x & size)) sh.list[x] = v, sh.list[y] = u;
              }
              __syncthreads();
            }
          // a thread's neighbouring places: their measure, and the last one before the target
          constexpr int L4 = kCap / kThreads;
          uint64_t ms[L4], sum = 0, whole;
#pragma unroll
          for (int i = 0; i < L4; i++) {
            const uint32_t x = tid * L4 + i;
            ms[i] = x < m ? (weigh ? fixed(sc.weight(logit_of(sh.list[x]))) : 1ull) : 0;
            sum += ms[i];
          }
          uint64_t from = above + block_before(sum, sh.red, &whole);
          const auto last_before = [&](uint64_t at, double until) {
            uint32_t last = 0;
#pragma unroll
            for (int i = 0; i < L4; i++) {
              const uint32_t x = tid * L4 + i;
              if (x < m && ((double)at < until || (lo == 0 && x == 0))) last = x + 1;
              at += ms[i];
            }
            return (uint32_t)block_max64(last, sh.red2);
          };
          uint32_t kept_n = last_before(from, target);
          const bool in = kept_n > 0 && (kept_n < m || (double)(above + whole) >= target || hi == last_bin);
          const bool finish = in && lo == 0;
          uint64_t s = 0;
          if (!weigh && by_weight && in) {   // the weight of what top-k left
            sum = 0;
#pragma unroll
            for (int i = 0; i < L4; i++) {
              const uint32_t x = tid * L4 + i;
              ms[i] = x < kept_n ? fixed(sc.weight(logit_of(sh.list[x]))) : 0;
              sum += ms[i];
            }
            from = block_before(sum, sh.red, &s);
            if (finish) {   // top-p over the same list
              m = kept_n;
              kept_n = last_before(from, (double)p * (double)s);
            }
          }
          if (tid == 0) {
            sh.missed = !in;
            sh.cut = in ? sh.list[kept_n - 1] : 0;
            sh.sum = s;
            sh.over = above;
            sh.done = finish;
          }
          if (finish) {   // the race over the list
            uint64_t best = 0, kept = 0;
            const float *row_noise = a.noise + b * a.ld_noise;
            for (uint32_t x = tid; x < kept_n; x += kThreads) {
              const uint64_t pl = sh.list[x];
              const float l = logit_of(pl), w1 = sc.weight(l);
              if (!(w1 >= min_p) && x) continue;
              kept += fixed(w1);
              const float s1 = sc.d(l) - logf(__ldg(row_noise + id_of(pl)));
              if (s1 > -INFINITY) best = max64(best, place(s1, id_of(pl)));
            }
            kept = block_sum64(kept, sh.red);
            best = block_max64(best, sh.red2);
            const int id = id_of(best ? best : top);
            for (uint32_t x = tid; x < kept_n; x += kThreads)
              if (id_of(sh.list[x]) == id) {
                a.tok[b] = id;
                if (a.logp) a.logp[b] = sc.d(logit_of(sh.list[x])) - logf((float)kept * 0x1p-40f);
              }
          }
        }
        cluster.sync();
        const bool done = first->done, missed = first->missed;
        const uint64_t new_cut = first->cut, sum = first->sum, exact_over = first->over;
        if (tid == 0) sh.n_list = 0;
        cluster.sync();   // CTA 0's words are free again, and its shared memory is not needed by others past here
        if (done) return;
        if (!missed) {
          bisect = false;
          cut = new_cut;
          if (!weigh && by_weight)
            total = sum + (lo > 0 ? weigh_all([&](float l, int) { return sc.bin(l) < lo; }) : 0);
          break;
        }
        // what lies before bin lo is known now
        guess = before + (float)((target - (double)exact_over) * (weigh ? 0x1p-40 : 1.0));
      }
      if (bisect) {
        // the largest number x with measure(places > x) >= target: the cut is the next one
        uint64_t x = 0;
        for (int bit = 63; bit >= 0; bit--) {
          const uint64_t mid = x | 1ull << bit;
          float over = 0.0f;
          uint32_t n_over = 0;
          each([&](float l, int i) {
            const uint64_t pl = place(l, begin + i);
            if (pl <= mid || pl < cut) return;
            if (weigh) over += sc.weight(l);
            else n_over++;
          });
          const uint64_t s = block_sum64(weigh ? fixed(over) : n_over, sh.red);
          if (tid == 0) sh.above = s;
          cluster.sync();
          if ((double)cluster_sum(peer->above) >= target) x = mid;
          cluster.sync();
        }
        cut = x >= top ? top : max64(cut, x + 1);
        if (!weigh && by_weight) total = weigh_all([&](float l, int i) { return place(l, begin + i) >= cut; });
      }
      if (!weigh) last_bin = sc.bin(logit_of(cut));
    }
  }

  // ---- the race over everything kept
  float kept = 0.0f, best = -INFINITY;
  int best_i = -1;
  const float lcut = cut > 1 ? logit_of(cut) : -FLT_MAX, inv = fminf(1.0f / T, 1e38f);
  const float *noise = a.noise + b * a.ld_noise + begin;
  const auto race = [&](float l, int i, float e) {
    const uint64_t pl = place(l, begin + i);
    if (pl < cut) return;
    const float w = sc.weight(l);
    if (!(w >= min_p) && pl != top) return;
    kept += w;
    // most ids lose by far: division and logarithm only for those near the best so far
    const float d = sc.below(l) * inv;
    if (d - __logf(e) < best - 0.01f + 1e-6f * d) return;
    const float s = sc.d(l) - logf(e);
    if (s > best) best = s, best_i = begin + i;
  };
  if (RESIDENT && a.noise_vec) {
    for (int i = tid; i < nv; i += kThreads) {
      const uint4 v = reinterpret_cast<const uint4 *>(held)[i];
      const In *x = reinterpret_cast<const In *>(&v);
      float4 e[E / 4];
      bool any[E / 4];
#pragma unroll
      for (int q = 0; q < E / 4; q++) {   // the random numbers of four ids where one of them is kept
        any[q] = false;
#pragma unroll
        for (int j = 0; j < 4; j++) any[q] |= to_float(x[4 * q + j]) >= lcut;
        const int at = i * E + 4 * q;
        if (any[q] && at + 4 <= n) e[q] = __ldg(reinterpret_cast<const float4 *>(noise + at));
        else if (any[q])
          e[q] = make_float4(at < n ? __ldg(noise + at) : 1.0f, at + 1 < n ? __ldg(noise + at + 1) : 1.0f,
                             at + 2 < n ? __ldg(noise + at + 2) : 1.0f, 1.0f);
      }
#pragma unroll
      for (int q = 0; q < E / 4; q++)
        if (any[q]) {
          const float ee[4] = {e[q].x, e[q].y, e[q].z, e[q].w};
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (to_float(x[4 * q + j]) >= lcut) race(to_float(x[4 * q + j]), i * E + 4 * q + j, ee[j]);
        }
    }
  } else {
    each([&](float l, int i) {
      if (l >= lcut && i < n) race(l, i, __ldg(noise + i));
    });
  }
  const uint64_t all = block_sum64(fixed(kept), sh.red);
  const uint64_t won = block_max64(best_i < 0 ? 0 : place(best, best_i), sh.red2);
  if (tid == 0) sh.kept = all, sh.best = won;
  cluster.sync();
  if (rank == 0 && tid < 32) {
    const uint64_t w = cluster_max(peer->best), sum = cluster_sum(peer->kept);
    const int id = id_of(w ? w : top);
    if (tid == 0) {
      a.tok[b] = id;
      if (a.logp) a.logp[b] = sc.d(to_float(static_cast<const In *>(a.logits)[b * a.ld + id])) - logf((float)sum * 0x1p-40f);
    }
  }
  cluster.sync();
}

template <typename In>
int launch(SampleParams p, int B, cudaStream_t st) {
  static int ready[64];
  int dev = 0, sms = 148;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev >= 64) return sm100_set_error(SM100_ERR_CUDA, "sample: device %d: %s", dev, cudaGetErrorString(e));
  constexpr int kHeld = 64 * 1024, kMost = 160 * 1024;   // two CTAs an SM; one where a row needs it
  if (!ready[dev]) {
    if ((e = cudaFuncSetAttribute(sample_kernel<In, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost)) != cudaSuccess)
      return sm100_set_error(SM100_ERR_CUDA, "sample: %s", cudaGetErrorString(e));
    ready[dev] = 1;
  }
  // CTAs of a row: what holds it, and more while the GPU is not full and a CTA has over 2048 ids
  int C = 1;
  while (C < kMaxCtas && ((int64_t)p.V * (int)sizeof(In) > (int64_t)C * kHeld || ((int64_t)B * C * 2 <= sms && p.V > 2048 * C))) C *= 2;
  p.chunk = ((p.V + C - 1) / C + 15) / 16 * 16;
  const size_t bytes = (size_t)p.chunk * sizeof(In);
  const bool resident = bytes <= kMost;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = resident ? bytes : 0;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  e = resident ? cudaLaunchKernelEx(&cfg, sample_kernel<In, true>, p) : cudaLaunchKernelEx(&cfg, sample_kernel<In, false>, p);
  if (e != cudaSuccess) return sm100_set_error(SM100_ERR_CUDA, "sample: %s", cudaGetErrorString(e));
  return launch_status("sample");
}

}  // namespace

extern "C" int sm100_sample(const Sm100SampleArgs *a, void *stream) {
  if (a && a->B == 0) return SM100_OK;
  if (!a || !a->logits || !a->noise || !a->tok || a->B < 0 || a->B > 1 << 24 || a->V < 1 || a->V >= 1 << 23 || a->ld < 0 ||
      a->ld_noise < 0 || (a->ld && a->ld < a->V) || (a->ld_noise && a->ld_noise < a->V))
    return sm100_set_error(SM100_ERR_ARG, "sample: B %d V %d (1 .. 2^23 - 1) ld %lld ld_noise %lld", a ? a->B : 0,
                           a ? a->V : 0, a ? (long long)a->ld : 0, a ? (long long)a->ld_noise : 0);
  if (a->dtype != SM100_DT_F32 && a->dtype != SM100_DT_BF16)
    return sm100_set_error(SM100_ERR_UNSUPPORTED, "sample: logits dtype %d (f32 or bf16)", a->dtype);
  SampleParams p{a->logits, a->noise, a->temperature, a->top_k, a->top_p, a->min_p, a->tok, a->logp,
                 a->ld ? a->ld : a->V, a->ld_noise ? a->ld_noise : a->V, a->V, 0, 0, 0};
  const int size = a->dtype == SM100_DT_F32 ? 4 : 2;
  p.vec = ((uintptr_t)a->logits & 15) == 0 && (a->B == 1 || p.ld * size % 16 == 0);
  p.noise_vec = ((uintptr_t)a->noise & 15) == 0 && (a->B == 1 || p.ld_noise % 4 == 0);
  return a->dtype == SM100_DT_F32 ? launch<float>(p, a->B, (cudaStream_t)stream)
                                  : launch<__nv_bfloat16>(p, a->B, (cudaStream_t)stream);
}
