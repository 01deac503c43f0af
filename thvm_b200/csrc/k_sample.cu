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
// What bounds it: the logits once (and the random numbers of the kept ids) is the
// floor; above it, with many rows the slowest row (256 x 102400 bf16: 79 to 93 us
// with the draw of the settings, 8 for the bytes, 33 instructions an id over all
// passes; a traced row takes 35 us on average, the longest 66), with few rows the
// latency of the steps one after the other (one row of 50257: 17 us, 32 of 102400:
// 30 to 34).  A row belongs to one CTA, or with few rows to a cluster of 2 to 8
// that holds it in shared memory where it fits (later passes come from L2
// otherwise).  A cut is found without sorting the row:
//   1. a histogram of (l_max - l) / T in 4096 bins of 1/128 of the ids that can
//      be chosen at all, summed over the cluster slice by slice;
//   2. the bins that can hold the cut: by count it is one; by weight a bin's
//      ids weigh count * e^-bin within e^(+-1/256), which bounds the cut to some
//      bins, and where those hold too many ids, narrower bounds about a guess
//      that knows the row's whole weight;
//   3. one pass gathers the ids of those bins (a few hundred), among which CTA 0
//      selects, sums what lies above them, which is kept, and runs its race; a
//      guess that missed is put right by what the pass summed.
// Where everything above the cut fits in the list too (top-k of up to some
// hundreds, a peaked top-p) the list is all that is kept, and CTA 0 runs the
// race on it alone.  A bin that overflows the list (thousands of equal logits at
// the cut) falls back to a bisection over the 64 bits of a place, a pass over the
// row for each: rows of one value take 185 to 200 us at 1 x 50257, 3.5 to 5.7 ms at 256
// x 102400.
// A thread sums the weights of its ids in f32, in a fixed order (V / 512 of them
// where one CTA has the row, 200 at 102400, fewer with more CTAs); from there on
// sums are 64-bit integers in units of 2^-40, so no order of arrival enters a
// result.  What a thread sums depends on the CTAs a row, and so on the batch: the
// totals of a row with 1, 2, 4 and 8 differ by some 2e-8 of it (emulated).  Whole
// numbers for every id would cost a conversion each, some 8 us when it was tried.
#include "common.cuh"
#include "sample_bins.h"

#include <cooperative_groups.h>
#include <float.h>

namespace cg = cooperative_groups;
using namespace sm100;

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 4096, kCap = 2048, kMost = 8;   // kMost: CTAs of a row
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

// the largest of 16 bytes of logits; NaN only where all are
__device__ __forceinline__ float largest(const uint4 &v, float) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
__device__ __forceinline__ float largest(const uint4 &v, __nv_bfloat16) {
  const __nv_bfloat162 *x = reinterpret_cast<const __nv_bfloat162 *>(&v);
  const __nv_bfloat162 m = __hmax2(__hmax2(x[0], x[1]), __hmax2(x[2], x[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// 0 for a logit that is left out
__device__ __forceinline__ uint64_t place(float l, int i) {
  if (!(l > -INFINITY)) return 0;
  l += 0.0f;   // -0 and 0 are equal logits
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

// The estimated weight of a bin's ids
__device__ __forceinline__ BinSum bin_weight(int bin, uint32_t ids) { return ids * fixed(__expf(-(float)bin / kPerNat)); }

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// -inf and NaN as -inf (left out), +inf as the largest float
__device__ __forceinline__ float clean(float l) { return fminf(fmaxf(l, -INFINITY), FLT_MAX); }

// A row's logits as weights and bins, a few instructions an id: w = 2^((l -
// l_max) * (log2(e) / T)), off by some 2^-22 and the product's rounding; bins of
// 1 / kPerNat around their multiples, the last one taking all that lies further.
struct Scale {
  float lmax, T, hi, per;
  __device__ void set(float top, float t) {
    lmax = top, T = t;
    hi = (float)fmin(1.4426950408889634 / (double)t, 1e38);
    per = fminf(kPerNat / t, 1e38f);
  }
  __device__ __forceinline__ float weight(float l) const {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"((l - lmax) * hi));
    return w;
  }
  __device__ __forceinline__ float bin_float(float l) const { return fmaf(lmax - l, per, 12582912.0f); }   // 1.5 * 2^23 + bin
  __device__ __forceinline__ int bin(float l) const {
    return __float_as_int(fminf(bin_float(l), 12582912.0f + (kBins - 1))) - 0x4b400000;
  }
  __device__ __forceinline__ float d(float l) const { return (l - lmax) / T; }
};

// adds 1 to the bin of a logit above a bound
__device__ __forceinline__ void count(uint32_t *bin, float l, float above) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.gt.f32 p, %1, %2;\n\t@p red.shared.add.u32 [%0], 1;\n\t}" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(bin)), "f"(l), "f"(above)
               : "memory");
}

// A sum reaches `goal` in bin `bin`; ids and estimated weight before the bin,
// ids up to its end.
struct Crossing {
  int bin;
  uint32_t before, upto;
  float weight_before;
};

enum { kSureLo, kSureHi, kWideLo, kWideHi, kNearLo, kNearHi, kGuess, kGoals, kLast = kGoals };

struct alignas(16) Shared {
  union {   // the histogram is in registers before the list begins
    uint64_t list[kCap];
    uint32_t hist[kBins];
  };
  uint32_t part_n[kThreads], part_lo[kThreads], part_hi[kThreads];   // select(): places, low and high 20 bits of measure
  uint64_t few[32], pick_over;
  uint32_t pick_n, n_few;
  uint64_t red[kWarps], red2[kWarps];
  uint32_t n_list;                 // gathered places
  Crossing cross[kGoals + 1];      // kLast: the last bin that matters
  // what each CTA of the cluster has pushed here: a push and a barrier are one hop, a read after the barrier another
  struct {
    uint64_t top, row, near, above, best, kept;   // largest place; weight of all ids, of those in the bins; measure above the
                                                  // list's bins; winner there and kept weight
    BinSum heavy;                                 // the slice's estimated weight
    uint32_t ids, n_list;                         // ids in its slice of bins; places on its list
  } from[kMost];
  uint64_t cut, sum, over;         // from CTA 0
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

// Of the list's places >= from: the last one whose forerunners measure less
// than target - over (`always` the first one), 0 where there is none; *upto:
// over and what is measured up to it, *all: over and all of them.  Places are
// spread over 512 bins between their ends until the bin of the cut has a warp's
// worth; the warps then compare those all with all, each for itself.
template <typename Measure>
__device__ uint64_t select(Shared &sh, uint32_t m, uint64_t from, uint64_t over, double target, bool always, Measure measure,
                           uint64_t *upto, uint64_t *all) {
  const int tid = threadIdx.x, lane = tid & 31;
  uint64_t a = from, b = ~0ull, first = 0;
  for (int level = 0;; level++) {
    uint64_t low = ~0ull, high = 0;
    for (uint32_t x = tid; x < m; x += kThreads) {
      const uint64_t pl = sh.list[x];
      if (pl >= a && pl <= b) low = pl < low ? pl : low, high = max64(high, pl);
    }
    b = block_max64(high, sh.red);
    a = ~block_max64(~low, sh.red2);
    if (level == 0) first = b;
    const int shift = max(0, 64 - 9 - (b == a ? 64 : __clzll((long long)(b - a))));
    sh.part_n[tid] = sh.part_lo[tid] = sh.part_hi[tid] = 0;
    if (tid == 0) sh.n_few = 0;
    __syncthreads();
    for (uint32_t x = tid; x < m; x += kThreads) {
      const uint64_t pl = sh.list[x];
      if (pl < a || pl > b) continue;
      const uint64_t v = measure(pl);
      const int bin = (int)((b - pl) >> shift);
      atomicAdd(&sh.part_n[bin], 1u);
      atomicAdd(&sh.part_lo[bin], (uint32_t)(v & 0xfffff));
      atomicAdd(&sh.part_hi[bin], (uint32_t)(v >> 20));
    }
    __syncthreads();
    uint64_t sum;
    const uint32_t n = sh.part_n[tid];
    const uint64_t before = over + block_before(((uint64_t)sh.part_hi[tid] << 20) + sh.part_lo[tid], sh.red, &sum);
    if (level == 0) *all = over + sum;
    const bool ok = n && ((double)before < target || (always && level == 0 && tid == 0));
    const int pick = (int)block_max64(ok ? tid + 1 : 0, sh.red2) - 1;
    if (pick < 0) return 0;
    if (tid == pick) sh.pick_over = before, sh.pick_n = n;
    b -= (uint64_t)pick << shift;
    a = max64(a, b - (1ull << shift) + 1);
    __syncthreads();
    over = sh.pick_over;
    if (sh.pick_n > 32) continue;
    for (uint32_t x = tid; x < m; x += kThreads) {
      const uint64_t pl = sh.list[x];
      if (pl >= a && pl <= b) sh.few[atomicAdd(&sh.n_few, 1u)] = pl;
    }
    __syncthreads();
    const int f = (int)sh.n_few;
    const uint64_t pl = lane < f ? sh.few[lane] : 0, v = lane < f ? measure(pl) : 0;
    uint64_t mine = over;
    for (int i = 0; i < f; i++) {
      const uint64_t other = __shfl_sync(0xffffffffu, pl, i), w = __shfl_sync(0xffffffffu, v, i);
      if (other > pl) mine += w;
    }
    uint64_t cut = lane < f && ((double)mine < target || (always && pl == first)) ? ~pl : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cut = max64(cut, __shfl_xor_sync(0xffffffffu, cut, o));
    const int who = __ffs(__ballot_sync(0xffffffffu, ~pl == cut && lane < f)) - 1;
    *upto = __shfl_sync(0xffffffffu, mine + v, max(who, 0));
    return cut ? ~cut : 0;
  }
}

template <typename In, bool RESIDENT, int C>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams a) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shared sh;
  constexpr int E = 16 / sizeof(In);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = C > 1 ? (int)cluster.block_rank() : 0, tid = threadIdx.x;
  const int b = blockIdx.x / C;
  pdl_trigger();
  if constexpr (C > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  for (int i = tid; i < kBins; i += kThreads) sh.hist[i] = 0;
  pdl_wait();
  const int begin = min(rank * a.chunk, a.V), n = min(a.V - begin, a.chunk);
  const In *src = static_cast<const In *>(a.logits) + b * a.ld + begin;
  In *held = reinterpret_cast<In *>(dyn);
  const auto sync = [&] {
    if constexpr (C > 1) cluster.sync();
    else __syncthreads();
  };
  // The CTA's ids as vectors of E neighbours, past the end -inf: in shared memory, or from L2 where the row does not fit; by
  // 16 bytes, or one by one where rows do not begin on 16 bytes
  const int nv = (n + E - 1) / E;
  const auto vector = [&](int i) {
    if (RESIDENT) return reinterpret_cast<const uint4 *>(held)[i];
    if (a.vec && (i + 1) * E <= n) return __ldg(reinterpret_cast<const uint4 *>(src) + i);
    uint4 v;
    In *y = reinterpret_cast<In *>(&v);
#pragma unroll
    for (int e = 0; e < E; e++) {
      if (i * E + e < n) y[e] = __ldg(src + i * E + e);
      else from_float(-INFINITY, y[e]);
    }
    return v;
  };
  // this thread's vectors in rising order, the next two under way
  const auto each_vector = [&](auto f) {
    uint4 v = tid < nv ? vector(tid) : uint4(), next = tid + kThreads < nv ? vector(tid + kThreads) : uint4();
#pragma unroll 1
    for (int i = tid; i < nv; i += kThreads) {
      const uint4 now = v;
      v = next;
      if (i + 2 * kThreads < nv) next = vector(i + 2 * kThreads);
      f(now, i);
    }
  };
  const float T = a.temperature ? a.temperature[b] : 1.0f;

  // ---- the row into shared memory, and its first place
  if constexpr (RESIDENT) {
    const int whole = a.vec ? n / E : 0;
#pragma unroll 4
    for (int i = tid; i < whole; i += kThreads)
      reinterpret_cast<uint4 *>(held)[i] = ld_stream_u4(src + (int64_t)i * E);
#pragma unroll 8
    for (int i = whole * E + tid; i < nv * E; i += kThreads) {
      if (i < n) held[i] = __ldg(src + i);
      else from_float(-INFINITY, held[i]);
    }
    __syncthreads();
  }
  float lmax = -INFINITY;
  int imax = 0;
#pragma unroll 4
  for (int i = tid; i < nv; i += kThreads) {
    const float x = clean(largest(vector(i), In()));   // +inf ties with the largest float
    if (x > lmax) lmax = x, imax = i * E;   // i rises: the first vector that holds the largest
  }
  const auto raw = [&](int i) { return to_float(RESIDENT ? held[i] : __ldg(src + i)); };
  uint64_t top = 0;
  if (lmax > -INFINITY) {   // the first of the vector
    for (int e = E - 1; e >= 0; e--)
      if (imax + e < n && clean(raw(imax + e)) == lmax) top = place(lmax, begin + imax + e);
  }
  top = block_max64(top, sh.red);
  if (tid == 0) sh.n_list = 0;
  if (tid <= kGoals) sh.cross[tid].bin = -1;
  if constexpr (C > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");   // every CTA has begun
  // the shared memory of CTA tid, for the threads that push a value to every CTA
  Shared *to = tid < C ? (C > 1 ? cluster.map_shared_rank(&sh, tid) : &sh) : nullptr;
  if (to) to->from[rank].top = top;
  sync();
  const auto *peer = &sh.from[(tid & 31) % C];   // the lanes of each warp take what every CTA has pushed
  const auto cluster_sum = [&](uint64_t v) {
    v = (tid & 31) < C ? v : 0;
#pragma unroll
    for (int o = C / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
  };
  const auto cluster_max = [&](uint64_t v) {
    v = (tid & 31) < C ? v : 0;
#pragma unroll
    for (int o = C / 2; o > 0; o >>= 1) v = max64(v, __shfl_xor_sync(0xffffffffu, v, o));
    return __shfl_sync(0xffffffffu, v, 0);
  };
  top = cluster_max(peer->top);
  const float min_p = a.min_p ? a.min_p[b] : 0.0f, p = a.top_p ? a.top_p[b] : 1.0f;
  if (top == 0 || !(T > 0.0f) || !(p > 0.0f) || !(min_p <= 1.0f)) {   // nothing, or the first id alone
    if (rank == 0 && tid == 0) {
      a.tok[b] = top == 0 ? -1 : id_of(top);
      if (a.logp) a.logp[b] = top == 0 ? -INFINITY : 0.0f;
    }
    return;
  }
  Scale sc;
  sc.set(logit_of(top), T);
  const bool wild = sc.lmax == FLT_MAX;   // there may be +inf among the logits
  const int k = a.top_k ? a.top_k[b] : 0;
  // a vector as floats; NaN stays (it fails every comparison below)
  const auto floats = [&](const uint4 &v, float x[E]) {
    const In *y = reinterpret_cast<const In *>(&v);
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = to_float(y[e]);
    if (wild) {
#pragma unroll
      for (int e = 0; e < E; e++) x[e] = clean(x[e]);
    }
  };
  // one id after the other, for what is rare
  const auto each = [&](auto f) {
    for (int i = tid; i < n; i += kThreads) f(clean(raw(i)), i);
  };
  // the measure of the cluster's places that pass a test
  const auto measure_all = [&](bool weigh, auto test) {
    float w = 0.0f;
    uint32_t c = 0;
    each([&](float l, int i) {
      const uint64_t pl = place(l, begin + i);
      if (pl == 0 || !test(l, pl)) return;
      if (weigh) w += sc.weight(l);
      else c++;
    });
    const uint64_t s = block_sum64(weigh ? fixed(w) : c, sh.red);
    if (to) to->from[rank].row = s;
    sync();
    const uint64_t all = cluster_sum(peer->row);
    sync();
    return all;
  };
  const float *noise = a.noise + b * a.ld_noise + begin;
  const float inv = fminf(1.0f / T, 1e38f);
  const auto score = [&](float l, int i) { return sc.d(l) - logf(__ldg(noise + i)); };
  const auto fast_score = [&](float l, float e) { return (l - sc.lmax) * inv - __logf(e); };
  const auto passes = [&](float l) { return sc.weight(l) >= min_p; };   // the first id's is 1

  uint64_t cut = 1, total = 0, near = 0;   // kept: place >= cut; what a top-p is a part of; of that what the bins hold
  bool past = false;
  bool by_count = k > 0 && k < a.V;
  const bool by_weight = p < 1.0f;
  int last_bin = kBins - 1;      // bins past it are cut off already
  constexpr int kB = kBins / C / kThreads;   // a CTA's slice of the bins, kB neighbours a thread
  const int bin0 = (rank * kThreads + tid) * kB;
  uint32_t cnt[kB], c_before = 0, valid = 0;
  BinSum w_before = 0;
  float unseen = 0.0f;   // the bins' weight beyond their estimate
  float l_far = -INFINITY;
#pragma unroll
  for (int i = 0; i < kB; i++) cnt[i] = 0;
  if (by_count || by_weight) {
    // ---- the histogram, and the weight of the row
    // Ids below a bound cannot be chosen and stay out of the histogram, whose scattered atomics are what this pass costs:
    // by weight alone those past x = -ln(V / (1 - p)) (together they weigh less than 1 - p of the first id, so top-p cuts
    // them whatever they are), and those that min-p leaves out, unless top-k's weight is top-p's whole
    float x_far = -INFINITY;
    if (!by_count && by_weight) x_far = -(logf((float)a.V) - logf(1.0f - p) + 0.1f);
    if (!(by_count && by_weight) && min_p > 0.0f) x_far = fmaxf(x_far, logf(fminf(min_p, 1.0f)) - 1e-3f);
    // (the last term: more than the roundings of the others, which are many nats where T is small beside l_max)
    const float below = x_far * T;
    l_far = fminf(sc.lmax + below - 0x1p-22f * (fabsf(sc.lmax) - below), nextafterf(sc.lmax, -INFINITY));
    float w = 0.0f, w_near = 0.0f;
    each_vector([&](const uint4 &v, int) {
      float x[E];
      floats(v, x);
      if (by_weight) {
#pragma unroll
        for (int e = 0; e < E; e++) w += x[e] > -INFINITY ? sc.weight(x[e]) : 0.0f;
      }
      if (largest(v, In()) > l_far) {
#pragma unroll
        for (int e = 0; e < E; e++) {
          count(&sh.hist[sc.bin(x[e])], x[e], l_far);
          if (by_weight) w_near += x[e] > l_far ? sc.weight(x[e]) : 0.0f;
        }
      }
    });
    if (by_weight) {
      const uint64_t s = block_sum64(fixed(w), sh.red), f = block_sum64(fixed(w_near), sh.red2);
      if (to) to->from[rank].row = s, to->from[rank].near = f;
    }
    sync();
    {
      uint32_t h[C][kB];
#pragma unroll
      for (int r = 0; r < C; r++) {
        const uint32_t *from = (C > 1 ? cluster.map_shared_rank(&sh, r) : &sh)->hist + bin0;
#pragma unroll
        for (int i = 0; i < kB; i++) h[r][i] = from[i];
      }
#pragma unroll
      for (int i = 0; i < kB; i++)
#pragma unroll
        for (int r = 0; r < C; r++) cnt[i] += h[r][i];
    }
    if (by_weight) {
      total = cluster_sum(peer->row);
      near = cluster_sum(peer->near);
    }
    uint32_t ids = 0;
    BinSum heavy = 0;
#pragma unroll
    for (int i = 0; i < kB; i++) ids += cnt[i], heavy += bin_weight(bin0 + i, cnt[i]);
    c_before = block_before(ids, reinterpret_cast<uint32_t *>(sh.red), &ids);
    w_before = block_before(heavy, sh.red2, &heavy);
    if (to) to->from[rank].ids = ids, to->from[rank].heavy = heavy;
    sync();
    const uint32_t c = (tid & 31) < C ? peer->ids : 0;
    const BinSum h = (tid & 31) < C ? peer->heavy : 0;
    BinSum all = 0;
#pragma unroll
    for (int r = 0; r < C; r++) {
      const uint32_t cr = __shfl_sync(0xffffffffu, c, r);
      const BinSum hr = __shfl_sync(0xffffffffu, h, r);
      if (r < rank) c_before += cr, w_before += hr;
      valid += cr, all += hr;
    }
    unseen = (float)(int64_t)(near - all) * 0x1p-40f;
    last_bin = sc.bin(l_far);
    if (by_weight && !by_count && (double)near < (double)p * (double)total) past = true;   // top-p cuts nothing that min-p leaves
    if (by_count && (uint32_t)k >= valid) by_count = false;   // top-k leaves every id there is
  }

  // round 0: top-k's cut, round 1: top-p's (or none): each finds its bins, gathers and selects; the last one runs the race
  for (int round = by_count ? 0 : 1; round < (by_weight || !by_count ? 2 : 1); round++) {
    const bool weigh = round == 1, filtered = weigh ? by_weight && !past : by_count, final_round = weigh || !by_weight;
    // the cut: the last place whose forerunners measure less than target
    const double target = weigh ? (double)p * (double)total : (double)k;
    const float goal = fmaxf((float)(target * (weigh ? 0x1p-40 : 1.0)), 1e-30f);
    // by weight a bin's estimate is within e^(1/256) of its weight.  The guess takes the row's whole weight as known and
    // estimates what lies past the cut: what is off there is the average of many light ids, not a few heavy ones
    float guess = weigh && !by_count ? goal - unseen : goal;
    bool bisect = true;
    for (int attempt = 0; attempt < 4; attempt++) {
      int lo = 0, hi = 0;
      float before = 0.0f;
      if (filtered) {
        {
          const float spread = weigh ? 1.0f : 0.0f;
          const auto sum_of = [&](float v) { return (BinSum)fmaxf(weigh ? v * 0x1p40f : v, 0.0f); };
          const BinSum goals[kGoals] = {sum_of(goal * (1.0f - 0.0045f * spread)), sum_of(goal * (1.0f + 0.0045f * spread)),
                                        sum_of(guess * (1.0f - 0.001f * spread)), sum_of(guess * (1.0f + 0.001f * spread)),
                                        sum_of(guess * (1.0f - 0.0002f * spread)), sum_of(guess * (1.0f + 0.0002f * spread)),
                                        sum_of(guess)};
          const auto tell = [&](int g, const Crossing &x) {
            for (int r = 0; r < C; r++) (C > 1 ? cluster.map_shared_rank(&sh, r) : &sh)->cross[g] = x;
          };
          uint32_t cc = c_before;
          BinSum ww = w_before;
#pragma unroll
          for (int i = 0; i < kB; i++) {
            if (bin0 + i == last_bin) tell(kLast, Crossing{last_bin, cc, cc + cnt[i], (float)ww * 0x1p-40f});
            if (cnt[i] == 0 || bin0 + i > last_bin) continue;
            const uint32_t c1 = cc + cnt[i];
            const BinSum w1 = ww + bin_weight(bin0 + i, cnt[i]);
#pragma unroll
            for (int g = 0; g < kGoals; g++)   // one thread of the cluster owns a goal
              if (reaches<BinSum>(weigh ? ww : cc, weigh ? w1 : c1, cc == 0, goals[g]))
                tell(g, Crossing{bin0 + i, cc, c1, (float)ww * 0x1p-40f});
            cc = c1, ww = w1;
          }
        }
        sync();
        // the widest bounds whose ids fit in the list; from the first id on, where those do
        bool fits = false;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          Crossing x = sh.cross[g < 3 ? 2 * g : kGuess], y = sh.cross[g < 3 ? 2 * g + 1 : kGuess];
          if (x.bin < 0) x = sh.cross[kLast];   // reached nowhere
          if (y.bin < 0) y = sh.cross[kLast];
          if (g == 0 && attempt) continue;   // the guess knows more by now
          if (fits) continue;
          if (y.upto <= kCap - 64) fits = true, lo = 0, before = 0.0f, hi = y.bin;
          else if (y.upto - x.before <= kCap - 64) fits = true, lo = x.bin, before = x.weight_before, hi = y.bin;
        }
        if (!fits) break;
      }
      // ---- the pass: ids above the bins are measured and, in the last round, race; those in the bins go on the list.  Of its
      // race a thread keeps the best two scores by fast math; what is within its error of the CTA's best is scored exactly
      // By logit: above x_lo is above the bins, down to x_hi on the list (a hundredth of a bin and some roundings more than the
      // bins hold; what the pass sums and gathers is what counts)
      const bool whole = filtered && lo == 0, racing = final_round && !whole;   // whole: the list holds all that is kept
      const float slack = 1e-6f * fabsf(sc.lmax);
      const float x_lo = !filtered ? l_far : whole ? INFINITY : sc.lmax - (lo - 0.51f) / sc.per * 0.999999f + slack;
      const float x_hi = !filtered ? INFINITY : hi == kBins - 1 ? -FLT_MAX : sc.lmax - (hi + 0.51f) / sc.per * 1.000001f - slack;
      const float x_any = fminf(x_lo, x_hi);   // below it a vector has nothing for this pass: most of a peaked row
      float over = 0.0f, kept = 0.0f, best = -INFINITY, second = -INFINITY;
      uint32_t n_over = 0;
      int best_i = -1;
      each_vector([&](const uint4 &v, int i) {
        const float most = largest(v, In());
        if (!(most >= x_any)) return;
        float x[E];
        floats(v, x);
        if (most > x_lo) {
          float e[E];
          if (racing) {
#pragma unroll
            for (int q = 0; q < E; q += 4) {   // the random numbers of four ids where one of them is kept
              e[q] = e[q + 1] = e[q + 2] = e[q + 3] = 1.0f;
              if (a.noise_vec && i * E + q + 4 <= n) {
                if (fmaxf(fmaxf(x[q], x[q + 1]), fmaxf(x[q + 2], x[q + 3])) > x_lo) {
                  const float4 r = __ldg(reinterpret_cast<const float4 *>(noise + i * E + q));
                  e[q] = r.x, e[q + 1] = r.y, e[q + 2] = r.z, e[q + 3] = r.w;
                }
              } else {
#pragma unroll
                for (int j = q; j < q + 4; j++)
                  if (x[j] > x_lo) e[j] = __ldg(noise + i * E + j);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < E; j++) {
            const bool up = x[j] > x_lo;
            const float w = up ? sc.weight(x[j]) : 0.0f;
            over += w;
            if (!weigh) n_over += up;
            if (racing) {
              const bool runs = up && w >= min_p;
              kept += runs ? w : 0.0f;
              const float f = runs ? fast_score(x[j], e[j]) : -INFINITY;
              second = fmaxf(second, fminf(f, best));
              if (f > best) best = f, best_i = i * E + j;
            }
          }
        }
        uint32_t in = 0;
#pragma unroll
        for (int e = 0; e < E; e++) in |= x[e] >= x_hi && x[e] <= x_lo ? 1u << e : 0u;
        while (in) {
          const int e = __ffs(in) - 1;
          in &= in - 1;
          float l = x[0];
#pragma unroll
          for (int j = 1; j < E; j++) l = j == e ? x[j] : l;
          const uint64_t pl = place(l, begin + i * E + e);
          if (pl < cut) continue;   // cut is at least 1: not the ids left out
          const uint32_t at = atomicAdd(&sh.n_list, 1u);
          if (at < kCap) sh.list[at] = pl;
        }
      });
      const uint64_t measured = whole ? 0 : block_sum64(weigh ? fixed(over) : n_over, sh.red);
      if (to) to->from[rank].above = measured;
      if (racing) {
        const uint64_t m = block_max64(best > -INFINITY ? place(clean(best), 0) : 0, sh.red2);
        const float from = logit_of(m) - 0.02f;
        uint64_t won = 0;
        const auto exact = [&](float l, int i) {
          const float s = score(l, i);
          if (s > -INFINITY) won = max64(won, place(clean(s), begin + i));
        };
        if (m != 0 && second >= from) {   // more than one of this thread's
          for (int i = tid; i < nv; i += kThreads)
            for (int j = i * E; j < min((i + 1) * E, n); j++) {
              const float l = clean(raw(j));
              if (l > x_lo && passes(l) && fast_score(l, __ldg(noise + j)) >= from) exact(l, j);
            }
        } else if (m != 0 && best >= from) {
          exact(clean(raw(best_i)), best_i);
        }
        won = block_max64(won, sh.red);
        const uint64_t sum = block_sum64(fixed(kept), sh.red2);
        if (to) to->from[rank].best = won, to->from[rank].kept = sum;
      }
      __syncthreads();
      if (to) to->from[rank].n_list = sh.n_list;
      sync();
      if (rank == 0) {
        // the other CTAs' places behind this one's
        const uint32_t c = (tid & 31) < C ? peer->n_list : 0;
        const uint64_t above = cluster_sum(peer->above);
        uint32_t m = __shfl_sync(0xffffffffu, c, 0);
#pragma unroll
        for (int r = 1; r < C; r++) {
          const uint32_t cr = __shfl_sync(0xffffffffu, c, r);
          for (uint32_t i = tid; i < cr && m + i < kCap; i += kThreads) sh.list[m + i] = cluster.map_shared_rank(&sh, r)->list[i];
          m += cr;
        }
        __syncthreads();
        uint64_t end = 0, upto, all = 0, s = 0;
        bool in = !filtered;
        if (filtered && m > 0 && m <= kCap) {   // ids past the histogram's bound can overflow the list
          // a measure is a weight, or 1 for each place
          const auto measure = [&](uint64_t pl) { return weigh ? fixed(sc.weight(logit_of(pl))) : 1ull; };
          end = select(sh, m, 0, above, target, whole, measure, &upto, &all);
          // the cut is in the list where what follows the list's last place is not kept
          in = end != 0 && (hi == last_bin || (double)all >= target);
        }
        if (!weigh && by_weight && in) {   // the weight of what top-k left
          const auto weight_of = [&](uint64_t pl) { return fixed(sc.weight(logit_of(pl))); };
          for (uint32_t x = tid; x < m; x += kThreads)
            if (sh.list[x] >= end) s += weight_of(sh.list[x]);
          s = block_sum64(s, sh.red);
          if (whole)   // top-p over the same list
            end = select(sh, m, end, 0, (double)p * (double)s, true, weight_of, &upto, &all);
        }
        const bool finish = in && (whole || final_round);
        if (to) {
          to->missed = !in;
          to->cut = end;
          to->sum = s;
          to->over = above;
          to->done = finish;
        }
        if (finish) {   // the race over the list, and the winners above it
          uint64_t best1 = 0, kept1 = 0;
          if (filtered)
            for (uint32_t x = tid; x < m; x += kThreads) {
              const uint64_t pl = sh.list[x];
              const float l = logit_of(pl), w1 = sc.weight(l);
              if (pl < end || !(w1 >= min_p)) continue;
              kept1 += fixed(w1);
              const float s1 = sc.d(l) - logf(__ldg(a.noise + b * a.ld_noise + id_of(pl)));
              if (s1 > -INFINITY) best1 = max64(best1, place(clean(s1), id_of(pl)));
            }
          kept1 = block_sum64(kept1, sh.red);
          best1 = block_max64(best1, sh.red2);
          if (racing) {
            kept1 += cluster_sum(peer->kept);
            best1 = max64(best1, cluster_max(peer->best));
          }
          if (tid == 0) {
            const int id = id_of(best1 ? best1 : top);
            a.tok[b] = id;
            if (a.logp) a.logp[b] = sc.d(clean(to_float(static_cast<const In *>(a.logits)[b * a.ld + id]))) - logf((float)kept1 * 0x1p-40f);
          }
        }
      }
      sync();
      if (sh.done) return;   // nothing reaches into another CTA past here
      const bool missed = sh.missed;
      const uint64_t new_cut = sh.cut, sum = sh.sum, exact_over = sh.over;
      if (tid == 0) sh.n_list = 0;
      if (tid <= kGoals) sh.cross[tid].bin = -1;
      sync();
      if (!missed) {
        bisect = false;
        cut = new_cut;
        if (!weigh && by_weight) total = sum + (lo > 0 ? measure_all(true, [&](float l, uint64_t) { return l > x_lo; }) : 0);
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
        if ((double)measure_all(weigh, [&](float, uint64_t pl) { return pl > mid && pl >= cut; }) >= target) x = mid;
      }
      cut = x >= top ? top : max64(cut, x + 1);
      if (!weigh && by_weight) total = measure_all(true, [&](float, uint64_t pl) { return pl >= cut; });
    }
    if (!weigh) last_bin = sc.bin(logit_of(cut));
  }

  // ---- the race over everything kept, where no list held the last cut
  float kept = 0.0f;
  uint64_t won = 0;
  each([&](float l, int i) {
    const uint64_t pl = place(l, begin + i);
    if (pl < cut || !passes(l)) return;
    kept += sc.weight(l);
    const float s = score(l, i);
    if (s > -INFINITY) won = max64(won, place(clean(s), begin + i));
  });
  const uint64_t all = block_sum64(fixed(kept), sh.red);
  won = block_max64(won, sh.red2);
  if (to) to->from[rank].kept = all, to->from[rank].best = won;
  sync();
  if (rank == 0 && tid < 32) {
    const uint64_t w = cluster_max(peer->best), sum = cluster_sum(peer->kept);
    const int id = id_of(w ? w : top);
    if (tid == 0) {
      a.tok[b] = id;
      if (a.logp) a.logp[b] = sc.d(clean(to_float(static_cast<const In *>(a.logits)[b * a.ld + id]))) - logf((float)sum * 0x1p-40f);
    }
  }
}

constexpr int kHeld = 64 * 1024;   // bytes of a row that a CTA holds: two CTAs an SM

// A launch of B clusters of C CTAs
template <typename In, bool RESIDENT, int C>
struct Launch {
  cudaLaunchAttribute at[2];
  cudaLaunchConfig_t cfg = {};
  Launch(int B, size_t dynamic, cudaStream_t st) {
    cfg.gridDim = dim3((unsigned)(B * C));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = dynamic;
    cfg.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = C;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = C > 1 ? 2 : 1;
  }
};

// Clusters of C CTAs that the device holds at once, asked for once a device (the largest shared memory that a launch takes);
// *e tells of a call that failed
template <typename In, bool RESIDENT, int C>
int clusters_at_once(cudaError_t *e) {
  static int known[64];   // clusters + 1
  const auto kernel = sample_kernel<In, RESIDENT, C>;
  int dev = 0, n = 0;
  if ((*e = cudaGetDevice(&dev)) != cudaSuccess) return 0;
  if (dev < 64 && known[dev]) return known[dev] - 1;
  if (RESIDENT && (*e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeld)) != cudaSuccess) return 0;
  Launch<In, RESIDENT, C> one(1, RESIDENT ? kHeld : 0, nullptr);
  one.at[0] = one.at[1];
  one.cfg.numAttrs = 1;
  if ((*e = cudaOccupancyMaxActiveClusters(&n, kernel, &one.cfg)) != cudaSuccess) return 0;
  if (dev < 64) known[dev] = n + 1;
  return n;
}

// C CTAs a row where a CTA's part is worth one and all rows run at once; *done tells whether it was launched
template <typename In, bool RESIDENT, int C>
cudaError_t launch_at_once(const SampleParams &p, int B, cudaStream_t st, bool *done) {
  cudaError_t e;
  if (B > clusters_at_once<In, RESIDENT, C>(&e) || e != cudaSuccess) return e;
  *done = true;
  Launch<In, RESIDENT, C> l(B, RESIDENT ? (p.chunk * sizeof(In) + 15) / 16 * 16 : 0, st);
  return cudaLaunchKernelEx(&l.cfg, sample_kernel<In, RESIDENT, C>, p);
}

template <typename In, int C>
cudaError_t try_row(SampleParams p, int B, cudaStream_t st, bool *done) {
  if (*done || p.V <= C * 1024) return cudaSuccess;
  p.chunk = ((p.V + C - 1) / C + 15) / 16 * 16;
  return p.chunk * (int64_t)sizeof(In) <= kHeld ? launch_at_once<In, true, C>(p, B, st, done)
                                                : launch_at_once<In, false, C>(p, B, st, done);
}

// CTAs of a row: as many as let every row run at once, up to 8.  A row's passes are bound by its SM, so more CTAs a row are
// faster until clusters have to wait for one another, which the GPU's groups of SMs decide: 8 fit up to 33 or 34 rows, 4 up to
// 70 or 71, 2 up to 148.  bf16 rows of 102400, top-k, with 1, 2, 4, 8 CTAs a row: 33 rows -, 29, 24, 24 us, 35 rows -, 30, 24, 38,
// 70 rows -, 34, 27, 58, 72 rows -, 33, 41, 59, 148 rows 34, 36, 67, -; rows of mixed settings differ in length, so that there
// 2 take 70 us at 148 rows where 1 takes 99.  Beyond, one CTA a row: 256 rows of top-p 82, 81, 95, 164.
template <typename In>
cudaError_t launch_row(SampleParams p, int B, cudaStream_t st) {
  bool done = false;
  cudaError_t e = try_row<In, 8>(p, B, st, &done);
  if (e == cudaSuccess) e = try_row<In, 4>(p, B, st, &done);
  if (e == cudaSuccess) e = try_row<In, 2>(p, B, st, &done);
  if (e != cudaSuccess || done) return e;
  p.chunk = (p.V + 15) / 16 * 16;
  Launch<In, false, 1> l(B, 0, st);
  return cudaLaunchKernelEx(&l.cfg, sample_kernel<In, false, 1>, p);
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
  const cudaError_t e = a->dtype == SM100_DT_F32 ? launch_row<float>(p, a->B, (cudaStream_t)stream)
                                                 : launch_row<__nv_bfloat16>(p, a->B, (cudaStream_t)stream);
  if (e != cudaSuccess) return sm100_set_error(SM100_ERR_CUDA, "sample: %s", cudaGetErrorString(e));
  return launch_status("sample");
}
