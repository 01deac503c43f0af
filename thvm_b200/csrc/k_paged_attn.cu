// Attention of new rows over the paged key / value cache: out = softmax(q k^T
// scale) v, query head h on key head h / (heads / kv_heads), row r of n on keys
// 0 .. kv_len - n + r.
//
// What bounds it: every key and value is read once for up to 16 query columns
// (the heads of a group times the new rows), so a decode step is bound by
// memory, and in 4 bits, where a token of 128 + 128 dimensions is 144 bytes, by
// issue slots next to it (unpacking, about one instruction a value).
//
// Split.  The tiles (TS tokens) of all units (sequence, key head, 16 query
// columns) form one line that is cut into gridDim equal pieces, one per CTA, so
// ragged lengths and one long sequence load every SM alike; the cut is found on
// the device from kv_len, so a captured graph follows it.  A unit cut between
// CTAs leaves parts (maximum, sum, unscaled output, f32) in the scratch; the
// CTA that arrives last at the unit's counter joins them in CTA order (no
// order of arrival enters the result).
//
// A CTA: one warp brings tiles in by bulk copies (a page of a key head is one
// contiguous block: one copy) through a ring of stages; NW warps take 16 of a
// tile's tokens each, with a running maximum and sum of their own, joined when
// the unit ends.
//
// A warp's 16 tokens: S^T = K Q^T and O^T += V^T P^T by mma.m16n8k16 with
// tokens, then dimensions, as the 16 rows and the query columns as the 8: no
// half of the tensor work is padding at 8 columns, softmax columns and output
// columns belong to the same threads, and P^T becomes the second operand by two
// movmatrix.  Dimensions (and the 16 rows of V^T) may be taken in any order that
// both operands share, so a lane's fragments are neighbouring values: 16-byte
// loads in bf16, whole code words in 4 bits.  (tcgen05 would want 128 rows of
// queries, and unpacked codes written back to shared memory.)
//
// 4 bits: a code c enters the products as an exact bf16 integer (128 + c in
// K, put together by one AND-OR; c - 8 in V).  A group's scale and minimum
// are applied outside: S = s * (Q . (128 + c)) + (m - 128 s) * sum Q per group of
// 64 dimensions, and p * s per token is V's weight, sum p (m + 8 s) its shift.
#include "paged.cuh"
#include "tma.cuh"

using namespace sm100;

namespace {

struct AttnParams {
  const __nv_bfloat16 *q;
  const int32_t *kv_len, *q_off;
  __nv_bfloat16 *out;
  float *parts;        // [gridDim][2] of kPart floats
  uint32_t *counters;  // [gridDim], zero between launches
  int64_t ld_q;
  int T, heads, group;
  float scale_log2;    // scale * log2(e)
};

constexpr int kMaxPieces = 148 * 4;   // CTAs of a launch at most

template <int HD, int BITS, int NT>
struct Shape {
  static constexpr int NW = BITS == 4 ? 8 : 4;                  // warps at the products
  static constexpr int TS = 16 * NW;                            // tokens of a tile
  static constexpr int TOKEN = BITS == 4 ? HD / 2 + HD / kGroup * 4 : 2 * HD;
  static constexpr int TILE = 2 * TS * TOKEN;                   // bytes of a tile
  static constexpr int NC = 8 * NT;                             // query columns
  static constexpr int CTAS = HD == 256 || (BITS == 4 && NT == 2) ? 1 : 2;   // per SM
  static constexpr int RING = HD == 256 ? 196608 : 98304;       // bytes for stages
  static constexpr int STAGES = RING / TILE > 8 ? 8 : RING / TILE;
  static constexpr int CHUNK = 16;                              // accumulators joined at a time
  static constexpr int ACC = HD / 16 * NT * 4;                  // accumulators of a thread
  static constexpr int PART = ACC * 32 + 2 * NC;                // floats of a unit's part
  static constexpr int RED = NW * CHUNK * 32 * 4;
  static constexpr int SMEM = STAGES * TILE + RED + 1024;
};

__device__ __forceinline__ void mma_bf16(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// P^T fragments of 8 tokens x 8 columns: this thread's two weights as bf16 hi +
// bf16 lo (16 bits of each weight enter the product)
__device__ __forceinline__ void split_weights(float w0, float w1, uint32_t &hi, uint32_t &lo) {
  const uint32_t h = pack2(w0, w1);
  hi = transpose8x8(h);
  lo = transpose8x8(pack2(w0 - bf16_lo(h), w1 - bf16_hi(h)));
}

// two codes of a word (bits 4 i and 4 i + 16) as bf16 128 + c
__device__ __forceinline__ uint32_t codes128(uint32_t w, int i) { return ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u; }
// the same as bf16 c - 8
__device__ __forceinline__ uint32_t codes8(uint32_t w, int i) {
  const uint32_t v = codes128(w, i);
  __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162 *>(&v);
  x = __hsub2(x, __floats2bfloat162_rn(136.0f, 136.0f));
  return *reinterpret_cast<const uint32_t *>(&x);
}

// The line of tiles, in the order (sequence, key head, column tile, token tile).
template <int TS, int NC>
struct Line {
  const AttnParams *a;
  const PagedView *c;
  int s, h, ct, n_ct, rows, first, len;   // the current unit
  int tiles, skip;                        // its tiles; how many lie before the piece

  __device__ __forceinline__ void load(int seq, int &r, int &f, int &l) const {
    f = a->q_off ? a->q_off[seq] : seq;
    r = a->q_off ? a->q_off[seq + 1] - f : 1;
    if (f < 0 || r < 0 || f > a->T - r) r = 0;   // rows outside q: none
    l = min(max(a->kv_len[seq], 0), c->max_pages * c->page);
  }
  __device__ __forceinline__ int columns(int r) const { return (r * a->group + NC - 1) / NC; }
  // keys that the last row of a column tile sees
  __device__ __forceinline__ int keys(int r, int l, int t) const {
    const int last = min(r * a->group, (t + 1) * NC) - 1;
    return l - r + last / a->group + 1;
  }
  __device__ __forceinline__ int unit_tiles(int r, int l, int t) const {
    const int k = keys(r, l, t);
    return k <= TS ? 1 : (k + TS - 1) / TS;   // a unit without keys still has its output to write
  }
  __device__ __forceinline__ int64_t seq_tiles(int seq) const {
    int r, f, l;
    int64_t n = 0;
    load(seq, r, f, l);
    for (int t = 0, e = columns(r); t < e; t++) n += unit_tiles(r, l, t);
    return n * c->kv_heads;
  }
  __device__ int64_t total(int lane) const {
    int64_t n = 0;
    for (int i = lane; i < c->n_seq; i += 32) n += seq_tiles(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
  }
  // the unit of tile w of the line (w < total)
  __device__ void seek(int64_t w, int lane) {
    int64_t before = 0;
    int base = 0;
    for (;; base += 32) {
      const int64_t n = base + lane < c->n_seq ? seq_tiles(base + lane) : 0;
      int64_t up = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + up > w);
      if (past) {
        const int at = __ffs(past) - 1;
        s = base + at;
        before += __shfl_sync(0xffffffffu, up - n, at);
        break;
      }
      before += __shfl_sync(0xffffffffu, up, 31);
    }
    load(s, rows, first, len);
    n_ct = columns(rows);
    int64_t left = w - before, per = 0;
    for (int t = 0; t < n_ct; t++) per += unit_tiles(rows, len, t);
    h = (int)(left / per);
    left -= h * per;
    ct = 0;
    while (left >= (tiles = unit_tiles(rows, len, ct))) left -= tiles, ct++;
    skip = (int)left;
  }
  __device__ __forceinline__ void next() {
    skip = 0;
    if (++ct == n_ct) {
      ct = 0;
      if (++h == c->kv_heads) {
        h = 0;
        do load(++s, rows, first, len);
        while (rows == 0);
        n_ct = columns(rows);
      }
    }
    tiles = unit_tiles(rows, len, ct);
  }
};

template <int HD, int BITS, int NT>
__global__ void __launch_bounds__(Shape<HD, BITS, NT>::NW * 32 + 32, Shape<HD, BITS, NT>::CTAS)
    paged_attn_kernel(const __grid_constant__ PagedView c, const __grid_constant__ AttnParams a) {
  using S = Shape<HD, BITS, NT>;
  constexpr int NW = S::NW, TS = S::TS, NC = S::NC, STAGES = S::STAGES, GR = HD / kGroup;
  extern __shared__ __align__(128) uint8_t smem[];
  float *red = reinterpret_cast<float *>(smem + STAGES * S::TILE);
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ uint16_t valid[STAGES][NW];
  __shared__ float wm[NW][NC], wl[NW][NC], um[NC], ul[NC];
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < STAGES; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NW);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  Line<TS, NC> line;
  line.a = &a;
  line.c = &c;
  const int64_t total = line.total(lane);
  const int G = (int)min((int64_t)gridDim.x, total), me = blockIdx.x;   // every piece holds a tile
  if (me >= G) return;
  const int64_t w0 = total * me / G, w1 = total * (me + 1) / G;
  line.seek(w0, lane);
  int64_t w = w0;
  uint32_t it = 0;   // tiles through the ring

  if (warp == NW) {
    // ---- the copies
    const int per = TS >> c.page_log2;            // pages of a tile
    const uint32_t block = c.block;
    const uint64_t pol = policy_evict_first();
    bool ok_ring = true;
    while (w < w1 && ok_ring) {
      const int end = (int)min((int64_t)line.tiles, line.skip + (w1 - w));
      for (int t = line.skip; t < end; t++, it++) {
        const int st = it % STAGES;
        const int slot = t * per + lane, key = slot << c.page_log2;
        int id = -1;
        bool want = lane < per && key < line.len;
        if (want) id = c.table[(int64_t)line.s * c.max_pages + slot];
        const bool ok = want && (unsigned)id < (unsigned)c.n_pages;
        if (want && !ok) atomicOr(&g_paged_status, SM100_DECODE_ERR_ARG);
        const uint32_t oks = __ballot_sync(0xffffffffu, ok);
        if (it >= STAGES && !mbar_wait(&empty[st], (it / STAGES - 1) & 1, &g_paged_status, false)) {
          ok_ring = false;
          break;
        }
        if (lane < NW) {
          const int base = t * TS + 16 * lane, n = min(max(line.len - base, 0), 16);
          valid[st][lane] = oks >> ((16 * lane) >> c.page_log2) & 1 ? (uint16_t)((1u << n) - 1) : 0;
        }
        __syncwarp();
        if (lane == 0) mbar_expect_tx(&full[st], __popc(oks) * block);
        __syncwarp();
        if (ok)
          bulk_g2s_hint(smem + st * S::TILE + lane * block,
                        c.pool + ((int64_t)id * c.kv_heads + line.h) * block, block, &full[st], pol);
      }
      w += end - line.skip;
      if (w < w1) line.next();
    }
    if (lane == 0 && me == 0) {   // lengths past the table were cut
      for (int s = 0; s < c.n_seq; s++)
        if (a.kv_len[s] > c.max_pages * c.page) atomicOr(&g_paged_status, SM100_DECODE_ERR_ARG);
    }
    return;
  }

  // ---- the products
  const int g = lane >> 2, cq = lane & 3;
  bool stalled = false;
  while (w < w1) {
    const int end = (int)min((int64_t)line.tiles, line.skip + (w1 - w));
    const int n_cols = min(NC, line.rows * a.group - line.ct * NC);
    // Q^T fragments: column g of each 8, this lane's dimensions
    uint32_t qf[NT][HD / 8];
    float qs[GR][NT][2];   // 4 bits: sum of a column's queries over a group (columns 2 cq, 2 cq + 1)
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int col = nt * 8 + g, at = line.ct * NC + col;
      const __nv_bfloat16 *src = a.q + (int64_t)(line.first + at / a.group) * a.ld_q +
                                 (int64_t)(line.h * a.group + at % a.group) * HD;
      uint4 v[HD / 32];
#pragma unroll
      for (int i = 0; i < HD / 32; i++) {
        const int d = BITS == 4 ? (i >> 1) * 64 + cq * 16 + (i & 1) * 8 : i * 32 + cq * 8;
        v[i] = col < n_cols ? __ldg(reinterpret_cast<const uint4 *>(src + d)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < HD / 32; i++) {
        if constexpr (BITS == 4) {   // pairs (0, 4), (1, 5), (2, 6), (3, 7), as the codes come
          qf[nt][4 * i] = __byte_perm(v[i].x, v[i].z, 0x5410);
          qf[nt][4 * i + 1] = __byte_perm(v[i].x, v[i].z, 0x7632);
          qf[nt][4 * i + 2] = __byte_perm(v[i].y, v[i].w, 0x5410);
          qf[nt][4 * i + 3] = __byte_perm(v[i].y, v[i].w, 0x7632);
        } else {
          qf[nt][4 * i] = v[i].x, qf[nt][4 * i + 1] = v[i].y, qf[nt][4 * i + 2] = v[i].z, qf[nt][4 * i + 3] = v[i].w;
        }
      }
      if constexpr (BITS == 4) {
#pragma unroll
        for (int gr = 0; gr < GR; gr++) {
          float s = 0.0f;
#pragma unroll
          for (int i = 8 * gr; i < 8 * gr + 8; i++) s += bf16_lo(qf[nt][i]) + bf16_hi(qf[nt][i]);
          s += __shfl_xor_sync(0xffffffffu, s, 1);
          s += __shfl_xor_sync(0xffffffffu, s, 2);
          qs[gr][nt][0] = __shfl_sync(0xffffffffu, s, 8 * cq);
          qs[gr][nt][1] = __shfl_sync(0xffffffffu, s, 8 * cq + 4);
        }
      }
    }
    // keys that this thread's columns see; the smallest of the unit's columns
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int col = nt * 8 + 2 * cq + e, at = line.ct * NC + col;
        lim[nt][e] = col < n_cols ? line.len - line.rows + at / a.group + 1 : 0;
      }
    const int row0 = line.ct * NC / a.group, row1 = (line.ct * NC + n_cols - 1) / a.group;
    const int lim_min = line.len - line.rows + row0 + 1;
    float o[GR * 4][NT][4], l[NT][2], m[NT][2], z[GR][NT][2];
#pragma unroll
    for (int i = 0; i < GR * 4; i++)
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[i][nt][e] = 0.0f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        l[nt][e] = 0.0f, m[nt][e] = -INFINITY;
#pragma unroll
        for (int gr = 0; gr < GR; gr++) z[gr][nt][e] = 0.0f;
      }

    for (int t = line.skip; t < end; t++, it++) {
      const int st = it % STAGES;
      if (!stalled) stalled = !mbar_wait(&full[st], (it / STAGES) & 1, &g_paged_status, false);
      const uint32_t bits = stalled ? 0 : valid[st][warp];
      const int key0 = t * TS + 16 * warp;
      if (bits != 0) {
        // this warp's tokens inside their page block
        const int page_in = (16 * warp) >> c.page_log2, row_in = (16 * warp) & (c.page - 1);
        const uint8_t *kb = smem + st * S::TILE + page_in * c.block, *vb = kb + c.block / 2;
        const bool edge = bits != 0xffffu || key0 + 16 > lim_min;
        float sc[NT][4];
        if constexpr (BITS == 4) {
          const uint8_t *km = kb + c.page * (HD / 2) + (row_in + g) * (GR * 4);
          kb += (row_in + g) * (HD / 2) + cq * 8;
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) sc[nt][e] = 0.0f;
#pragma unroll
          for (int gr = 0; gr < GR; gr++) {
            const uint2 w0 = *reinterpret_cast<const uint2 *>(kb + gr * 32);
            const uint2 w8 = *reinterpret_cast<const uint2 *>(kb + gr * 32 + 8 * (HD / 2));
            const uint32_t m0 = *reinterpret_cast<const uint32_t *>(km + gr * 4);
            const uint32_t m8 = *reinterpret_cast<const uint32_t *>(km + gr * 4 + 8 * (GR * 4));
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
              for (int e = 0; e < 4; e++) acc[nt][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t x0 = i < 2 ? w0.x : w0.y, x8 = i < 2 ? w8.x : w8.y;
              const int j = 2 * (i & 1);
              const uint32_t af[4] = {codes128(x0, j), codes128(x8, j), codes128(x0, j + 1), codes128(x8, j + 1)};
#pragma unroll
              for (int nt = 0; nt < NT; nt++) mma_bf16(acc[nt], af, qf[nt][8 * gr + 2 * i], qf[nt][8 * gr + 2 * i + 1]);
            }
            const float s0 = bf16_lo(m0), s8 = bf16_lo(m8);
            const float b0 = fmaf(-128.0f, s0, bf16_hi(m0)), b8 = fmaf(-128.0f, s8, bf16_hi(m8));
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                sc[nt][e] = fmaf(s0, acc[nt][e], fmaf(b0, qs[gr][nt][e], sc[nt][e]));
                sc[nt][2 + e] = fmaf(s8, acc[nt][2 + e], fmaf(b8, qs[gr][nt][e], sc[nt][2 + e]));
              }
          }
        } else {
          kb += (row_in + g) * (2 * HD) + cq * 16;
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) sc[nt][e] = 0.0f;
#pragma unroll
          for (int i = 0; i < HD / 32; i++) {
            const uint4 x0 = *reinterpret_cast<const uint4 *>(kb + i * 64);
            const uint4 x8 = *reinterpret_cast<const uint4 *>(kb + i * 64 + 8 * (2 * HD));
            const uint32_t a0[4] = {x0.x, x8.x, x0.y, x8.y}, a1[4] = {x0.z, x8.z, x0.w, x8.w};
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              mma_bf16(sc[nt], a0, qf[nt][4 * i], qf[nt][4 * i + 1]);
              mma_bf16(sc[nt], a1, qf[nt][4 * i + 2], qf[nt][4 * i + 3]);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[nt][e] *= a.scale_log2;
        if (edge) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int r = e < 2 ? g : g + 8;
              if (!(bits >> r & 1) || key0 + r >= lim[nt][e & 1]) sc[nt][e] = -INFINITY;
            }
        }
        // the running maximum moves only where a column grows past it by 2^8 (a weight of up to 2^8 costs an f32 sum
        // nothing): most tiles then skip the reduction and the rescaling
        bool grows = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) grows |= fmaxf(sc[nt][e], sc[nt][2 + e]) > m[nt][e] + 8.0f;
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float v = fmaxf(fmaxf(sc[nt][e], sc[nt][2 + e]), m[nt][e]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
              const float f = v == -INFINITY ? 1.0f : ex2(m[nt][e] - v);
              m[nt][e] = v;
              l[nt][e] *= f;
#pragma unroll
              for (int gr = 0; gr < GR; gr++) z[gr][nt][e] *= f;
#pragma unroll
              for (int i = 0; i < GR * 4; i++) o[i][nt][e] *= f, o[i][nt][2 + e] *= f;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float mm = m[nt][e] == -INFINITY ? 0.0f : m[nt][e];
            sc[nt][e] = ex2(sc[nt][e] - mm);
            sc[nt][2 + e] = ex2(sc[nt][2 + e] - mm);
            l[nt][e] += sc[nt][e] + sc[nt][2 + e];
          }
        const int k0 = 2 * cq;   // this lane's tokens of V^T: k0, k0 + 1, k0 + 8, k0 + 9
        if constexpr (BITS == 4) {
          const uint8_t *vm = vb + c.page * (HD / 2) + (row_in + g) * (GR * 4);
          vb += (row_in + k0) * (HD / 2) + g * 4;
#pragma unroll
          for (int gr = 0; gr < GR; gr++) {
            const uint32_t m0 = *reinterpret_cast<const uint32_t *>(vm + gr * 4);
            const uint32_t m8 = *reinterpret_cast<const uint32_t *>(vm + gr * 4 + 8 * (GR * 4));
            float s0 = bf16_lo(m0), s8 = bf16_lo(m8);
            float b0 = fmaf(8.0f, s0, bf16_hi(m0)), b8 = fmaf(8.0f, s8, bf16_hi(m8));
            uint32_t p0[NT], p8[NT], r0[NT], r8[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              float w[4];
#pragma unroll
              for (int e = 0; e < 2; e++) {
                w[e] = sc[nt][e] * s0, w[2 + e] = sc[nt][2 + e] * s8;
                float d0 = sc[nt][e] * b0, d8 = sc[nt][2 + e] * b8;
                if (edge) {   // a weight of zero leaves out whatever the token holds
                  if (sc[nt][e] == 0.0f) w[e] = d0 = 0.0f;
                  if (sc[nt][2 + e] == 0.0f) w[2 + e] = d8 = 0.0f;
                }
                z[gr][nt][e] += d0 + d8;
              }
              split_weights(w[0], w[1], p0[nt], r0[nt]);
              split_weights(w[2], w[3], p8[nt], r8[nt]);
            }
            const uint32_t wa = *reinterpret_cast<const uint32_t *>(vb + gr * 32);
            const uint32_t wb = *reinterpret_cast<const uint32_t *>(vb + gr * 32 + (HD / 2));
            const uint32_t wc = *reinterpret_cast<const uint32_t *>(vb + gr * 32 + 8 * (HD / 2));
            const uint32_t wd = *reinterpret_cast<const uint32_t *>(vb + gr * 32 + 9 * (HD / 2));
            const uint32_t lo[2] = {__byte_perm(wa, wb, 0x5410), __byte_perm(wa, wb, 0x7632)};
            const uint32_t hi[2] = {__byte_perm(wc, wd, 0x5410), __byte_perm(wc, wd, 0x7632)};
#pragma unroll
            for (int j = 0; j < 4; j++) {   // dimensions 8 g + 2 j, 8 g + 2 j + 1 of the group
              const int i = 2 * (j & 1);
              const uint32_t af[4] = {codes8(lo[j >> 1], i), codes8(lo[j >> 1], i + 1), codes8(hi[j >> 1], i),
                                      codes8(hi[j >> 1], i + 1)};
#pragma unroll
              for (int nt = 0; nt < NT; nt++) {
                mma_bf16(o[4 * gr + j][nt], af, p0[nt], p8[nt]);
                mma_bf16(o[4 * gr + j][nt], af, r0[nt], r8[nt]);
              }
            }
          }
        } else {
          uint32_t p0[NT], p8[NT], r0[NT], r8[NT];
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            split_weights(sc[nt][0], sc[nt][1], p0[nt], r0[nt]);
            split_weights(sc[nt][2], sc[nt][3], p8[nt], r8[nt]);
          }
          vb += (row_in + k0) * (2 * HD) + g * 16;
          const int tk[4] = {k0, k0 + 1, k0 + 8, k0 + 9};
#pragma unroll
          for (int gr = 0; gr < GR; gr++) {
            uint4 x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = *reinterpret_cast<const uint4 *>(vb + gr * 128 + (tk[k] - k0) * (2 * HD));
            if (!edge) {
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const uint32_t wa = (&x[0].x)[j], wb = (&x[1].x)[j], wc = (&x[2].x)[j], wd = (&x[3].x)[j];
                const uint32_t af[4] = {__byte_perm(wa, wb, 0x5410), __byte_perm(wa, wb, 0x7632),
                                        __byte_perm(wc, wd, 0x5410), __byte_perm(wc, wd, 0x7632)};
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                  mma_bf16(o[4 * gr + j][nt], af, p0[nt], p8[nt]);
                  mma_bf16(o[4 * gr + j][nt], af, r0[nt], r8[nt]);
                }
              }
            } else {
              // row by row: a token that a row does not see is zeros to it, and another row's product, where that
              // token may hold an infinity or a NaN, does not enter its columns
              for (int r = row0; r <= row1; r++) {
                const int seen = line.len - line.rows + r + 1;
                uint32_t keep[4];
#pragma unroll
                for (int k = 0; k < 4; k++) keep[k] = (bits >> tk[k] & 1) && key0 + tk[k] < seen ? 0xffffffffu : 0u;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  const uint32_t wa = (&x[0].x)[j] & keep[0], wb = (&x[1].x)[j] & keep[1];
                  const uint32_t wc = (&x[2].x)[j] & keep[2], wd = (&x[3].x)[j] & keep[3];
                  const uint32_t af[4] = {__byte_perm(wa, wb, 0x5410), __byte_perm(wa, wb, 0x7632),
                                          __byte_perm(wc, wd, 0x5410), __byte_perm(wc, wd, 0x7632)};
#pragma unroll
                  for (int nt = 0; nt < NT; nt++) {
                    float tmp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_bf16(tmp, af, p0[nt], p8[nt]);
                    mma_bf16(tmp, af, r0[nt], r8[nt]);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                      if (lim[nt][e & 1] == seen) o[4 * gr + j][nt][e] += tmp[e];
                  }
                }
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }

    // ---- the warps' parts of the unit joined
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
          if constexpr (BITS == 4) {
#pragma unroll
            for (int gr = 0; gr < GR; gr++) z[gr][nt][e] += __shfl_xor_sync(0xffffffffu, z[gr][nt][e], x);
          }
        }
        if (g == 0) wm[warp][nt * 8 + 2 * cq + e] = m[nt][e], wl[warp][nt * 8 + 2 * cq + e] = l[nt][e];
      }
    const auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(NW * 32) : "memory"); };
    sync();
    float f[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int col = nt * 8 + 2 * cq + e;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; i++) top = fmaxf(top, wm[i][col]);
#pragma unroll
        for (int i = 0; i < NW; i++) sum += wm[i][col] == -INFINITY ? 0.0f : wl[i][col] * ex2(wm[i][col] - top);
        f[nt][e] = m[nt][e] == -INFINITY ? 0.0f : ex2(m[nt][e] - top);
        if (warp == 0 && g == 0) um[col] = top, ul[col] = sum;
      }
    // where the piece ends inside the unit, or began inside it: a part
    const bool whole = line.skip == 0 && end == line.tiles;
    float *part = a.parts + ((int64_t)me * 2 + (line.skip == 0)) * S::PART;
      const auto put = [&](int i, int nt, int e, float v0, float v1) {   // dimensions d, d + 1 of a column
      const int col = nt * 8 + 2 * cq + e, at = line.ct * NC + col;
      if (col >= n_cols) return;
      const int d = (i >> 2) * 64 + 8 * g + 2 * (i & 3);
      const float inv = ul[col] > 0.0f ? 1.0f / ul[col] : ul[col] == 0.0f ? 0.0f : ul[col];
      *reinterpret_cast<uint32_t *>(a.out + ((int64_t)(line.first + at / a.group) * a.heads + line.h * a.group + at % a.group) * HD + d) =
          pack2(v0 * inv, v1 * inv);
    };
    constexpr int CI = S::CHUNK / (4 * NT);   // accumulator tiles of a chunk
#pragma unroll
    for (int ch = 0; ch < GR * 4 / CI; ch++) {
#pragma unroll
      for (int k = 0; k < CI; k++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int i = ch * CI + k;
            float v = o[i][nt][e];
            if constexpr (BITS == 4) v += z[i >> 2][nt][e & 1];
            v = f[nt][e & 1] == 0.0f ? 0.0f : v * f[nt][e & 1];
            red[(warp * S::CHUNK + (k * NT + nt) * 4 + e) * 32 + lane] = v;
          }
      sync();
      // pairs of accumulators (e, e + 2), two neighbouring dimensions of a column, over the warps
#pragma unroll
      for (int y = 0; y < S::CHUNK / 2 / NW + (S::CHUNK / 2 % NW != 0); y++) {
        const int pr = y * NW + warp;
        if (pr < S::CHUNK / 2) {
          const int e = pr & 1, tile = pr >> 1, k = tile / NT, nt = tile % NT;
          float v0 = 0.0f, v1 = 0.0f;
#pragma unroll
          for (int x = 0; x < NW; x++) {
            v0 += red[(x * S::CHUNK + tile * 4 + e) * 32 + lane];
            v1 += red[(x * S::CHUNK + tile * 4 + e + 2) * 32 + lane];
          }
          if (whole) {
            put(ch * CI + k, nt, e, v0, v1);
          } else {
            const int at = (ch * (S::CHUNK / 2) + pr) * 64 + lane * 2;
            __stcg(reinterpret_cast<float2 *>(part + at), make_float2(v0, v1));
          }
        }
      }
      sync();
    }
    if (!whole) {
      if (tid < NC) {
        __stcg(part + S::ACC * 32 + tid, um[tid]);
        __stcg(part + S::ACC * 32 + NC + tid, ul[tid]);
      }
      // the CTAs that share the unit, by the line's positions of its first and last tile
      const int64_t u0 = w - line.skip, u1 = u0 + line.tiles - 1;
      const int c0 = (int)(((u0 + 1) * G - 1) / total), c1 = (int)(((u1 + 1) * G - 1) / total);
      __threadfence();
      sync();
      if (tid == 0) arrived = atomicAdd(&a.counters[c0], 1u);
      sync();
      if (arrived == (uint32_t)(c1 - c0)) {
        __threadfence();
        if (tid == 0) a.counters[c0] = 0;
        const float *base = a.parts;
        const auto part_of = [&](int x) { return base + ((int64_t)x * 2 + (x == c0)) * S::PART; };
        if (tid < NC) {
          float top = -INFINITY, sum = 0.0f;
          for (int x = c0; x <= c1; x++) {
            const float pm = __ldcg(part_of(x) + S::ACC * 32 + tid), pl = __ldcg(part_of(x) + S::ACC * 32 + NC + tid);
            if (pm == -INFINITY) continue;
            const float t = fmaxf(top, pm);
            sum = sum * ex2(top - t) + pl * ex2(pm - t);
            top = t;
          }
          um[tid] = top, ul[tid] = sum;
        }
        sync();
        for (int pr = warp; pr < S::ACC / 2; pr += NW) {
          const int e = pr & 1, nt = (pr >> 1) % NT, i = (pr >> 1) / NT;
          const int col = nt * 8 + 2 * cq + e;
          const float top = um[col];
          float v0 = 0.0f, v1 = 0.0f;
#pragma unroll 4
          for (int x = c0; x <= c1; x++) {
            const float *p = part_of(x);
            const float pm = __ldcg(p + S::ACC * 32 + col);
            const float2 v = __ldcg(reinterpret_cast<const float2 *>(p + pr * 64 + lane * 2));
            const float fx = pm == -INFINITY ? 0.0f : ex2(pm - top);
            if (fx != 0.0f) v0 += v.x * fx, v1 += v.y * fx;
          }
          put(i, nt, e, v0, v1);
        }
      }
      sync();
    }
    w += end - line.skip;
    if (w < w1) line.next();
  }
  if (stalled && warp == 0)   // a wait gave up: the copies still under way may not outlive the CTA's shared memory
    for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; i++)
      mbar_wait(&full[i % STAGES], (i / STAGES) & 1, &g_paged_status, false);
}

template <int HD, int BITS, int NT>
int launch(const PagedView &v, AttnParams &p, const Sm100PagedAttnArgs *a, cudaStream_t st) {
  using S = Shape<HD, BITS, NT>;
  static int grid[64];   // CTAs that one device holds at once, by ordinal
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev >= 64) return sm100_set_error(SM100_ERR_CUDA, "paged_attention: device %d: %s", dev, cudaGetErrorString(e));
  const auto kernel = paged_attn_kernel<HD, BITS, NT>;
  if (!grid[dev]) {
    int sms = 0, per = 0;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM)) != cudaSuccess ||
        (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess ||
        (e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, S::NW * 32 + 32, S::SMEM)) != cudaSuccess)
      return sm100_set_error(SM100_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
    if (per < 1) return sm100_set_error(SM100_ERR_UNSUPPORTED, "paged_attention: no room for %d bytes of shared memory", S::SMEM);
    grid[dev] = sms * per < kMaxPieces ? sms * per : kMaxPieces;
  }
  p.counters = static_cast<uint32_t *>(a->ws);
  p.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(a->ws) + kMaxPieces * 4);
  e = launch_pdl(kernel, dim3(grid[dev]), dim3(S::NW * 32 + 32), S::SMEM, st, v, p);
  if (e != cudaSuccess) return sm100_set_error(SM100_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
  return launch_status("paged_attention");
}

template <int HD, int BITS>
int launch_columns(const PagedView &v, AttnParams &p, const Sm100PagedAttnArgs *a, cudaStream_t st) {
  if constexpr (HD <= 128) {
    if ((int64_t)a->max_rows * p.group > 8) return launch<HD, BITS, 2>(v, p, a, st);
  }
  return launch<HD, BITS, 1>(v, p, a, st);
}

}  // namespace

extern "C" uint64_t sm100_paged_attention_ws_bytes(const Sm100PagedCache *c, int32_t heads, int32_t max_rows) {
  PagedView v;
  if (sm100_paged_view(c, "paged_attention_ws_bytes", &v) || heads < 1 || heads % c->kv_heads || max_rows < 1) return 0;
  const uint64_t cols = (uint64_t)max_rows * (heads / c->kv_heads) > 8 && c->head_dim <= 128 ? 16 : 8;
  return kMaxPieces * 4 + (uint64_t)kMaxPieces * 2 * (cols * c->head_dim + 2 * cols) * 4;
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
  if ((int64_t)a->T * a->heads / c->kv_heads > INT32_MAX)
    return sm100_set_error(SM100_ERR_ARG, "paged_attention: %d rows in one call", a->T);
  AttnParams p{static_cast<const __nv_bfloat16 *>(a->q), a->kv_len, a->q_off, static_cast<__nv_bfloat16 *>(a->out),
               nullptr, nullptr, ld, a->T, a->heads, a->heads / c->kv_heads, a->scale * 1.4426950408889634f};
  cudaStream_t st = (cudaStream_t)stream;
  const bool q4 = c->bits == SM100_KV_Q4;
  if (c->head_dim == 64) return q4 ? launch_columns<64, 4>(v, p, a, st) : launch_columns<64, 16>(v, p, a, st);
  if (c->head_dim == 128) return q4 ? launch_columns<128, 4>(v, p, a, st) : launch_columns<128, 16>(v, p, a, st);
  return q4 ? launch_columns<256, 4>(v, p, a, st) : launch_columns<256, 16>(v, p, a, st);
}

uint32_t sm100_paged_attn_take_status(void) {
  uint32_t v = 0, z = 0;
  cudaMemcpyFromSymbol(&v, g_paged_status, sizeof(v));
  cudaMemcpyToSymbol(g_paged_status, &z, sizeof(z));
  return v;
}
