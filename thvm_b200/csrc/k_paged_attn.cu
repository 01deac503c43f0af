// Attention of new rows over the paged key / value cache: out = softmax(q k^T
// scale) v, query head h on key head h / (heads / kv_heads), row r of n on keys
// 0 .. kv_len - n + r.
//
// What bounds it: every key and value is read once for up to 8 query columns
// (the heads of a group times the new rows), so a decode step is bound by
// memory: bf16 pages stream at 5.5 TB/s (16 sequences of 4096, 8 key heads of
// 128: 49 us).  In 4 bits, where a token of 128 + 128 dimensions is 144 bytes,
// issue and the integer pipe bind first: of the 369 instructions for 16 tokens
// 136 are the shifts and ANDs that unpack (16 sequences of 16384: 57 % of the
// issue slots and 58 % of the integer pipe, memory at 42 %; 64 of up to 16384:
// 137 to 141 us, 3.8 TB/s).  Short calls are bound by the chain lengths -> cut -> table
// -> first tile and by the joining (one sequence of 32768 in 4 bits, 24 us: tiles
// done after 7 to 15, the last unit joined 10 later).
//
// Split.  The tiles (TS tokens) of all units (sequence, key head, 8 query
// columns) form one line that is cut into gridDim equal pieces, one per CTA, so
// ragged lengths and one long sequence load every SM alike; the cut is found on
// the device from kv_len, so a captured graph follows it.  A unit cut between
// CTAs leaves parts (maximum, sum, unscaled output, f32) in the scratch; the
// CTA that arrives last at the unit's counter joins them in CTA order (no
// order of arrival enters the result).
//
// A CTA: one warp brings tiles in by bulk copies (a page's keys, values and
// their marks, each area of the tile's pages end to end, so that every place in
// a tile is a constant) through a ring of stages; four warps take a quarter of a
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
// 4 bits: a code c enters the products as an exact bf16 integer (128 + c in K;
// in V 16 + c for tokens 0 .. 7 of 16 and c - 31 = -(16 + (15 - c)) for the
// others), put together by a shift and one three-input logic operation, a known
// way to make numbers of codes.  A group's scale and minimum are applied outside:
// S = s * (Q . (128 + c)) + (m - 128 s) * sum Q per group of 64 dimensions, and
// p * s per token is V's weight, sum p (m - 16 s) or p (m + 31 s) its shift.  The
// products round their running sums towards zero: with one sign for all tokens
// the sums of 16 + c grew to some 20 times the output, and long ones leaned by
// 2^-13 of the mean |v|; with two signs they stay near zero (64 x up to 16384: 17 % of
// the outputs were a bf16 step off the rounded result, 1.4 % are, in the same time).
// Weights enter as bf16 hi + lo, so their rounding (2^-17) is far below the
// output's; with up to 4 query columns the low parts are columns 4 to 7 of the
// same product.
#include <float.h>

#include "paged.cuh"
#include "tma.cuh"

using namespace sm100;

namespace {

struct AttnParams {
  const __nv_bfloat16 *q;
  const int32_t *kv_len, *q_off;
  __nv_bfloat16 *out;
  float *parts;        // [gridDim][2] of Shape::PART floats
  uint32_t *counters;  // [gridDim], zero between launches
  int64_t ld_q;
  int T, heads, group;
  float scale_log2;    // scale * log2(e)
};

constexpr int kSMs = 148;

// CTAs of an SM: what the registers leave (5 warps each: 128 registers at 3, 168 at 2, 255 at 1)
constexpr int ctas_of(int hd, int bits) { return hd == 256 ? (bits == 4 ? 2 : 1) : hd == 128 && bits == 16 ? 2 : 3; }

constexpr int kCounters = kSMs * 4;   // the most CTAs of a launch are 3 an SM

// COLS query columns a unit: 4 (4 bits only: the weights' low parts take the
// other half of the 8 columns of a product) or 8.  Two products a unit, 16
// columns, unpack a token once for both but leave registers for two CTAs an SM
// only: 8 x 4096 tokens in 4 bits with 32 columns a key head took 40 us, 34.5 in
// units of 8.
template <int HD, int BITS, int COLS>
struct Shape {
  static constexpr int NW = 4;                                  // warps at the products
  static constexpr int KS = BITS == 4 || HD == 64 ? 2 : 1;      // 16-token steps that a warp takes of a tile
  static constexpr int TS = 16 * KS * NW;                       // tokens of a tile
  static constexpr int GR = HD / kGroup;
  static constexpr int ROW = BITS == 4 ? HD / 2 : 2 * HD;       // bytes of a token's keys
  static constexpr int MARKS = BITS == 4 ? 4 * GR : 0;          // and of their scales and minima
  // a tile in shared memory: keys, their marks, values, their marks of all tokens
  static constexpr int V = TS * (ROW + MARKS), TILE = 2 * V;
  static constexpr bool DUAL = COLS == 4;
  static constexpr int ACC = HD / 16;                           // accumulator tiles (4 floats) of a thread
  static constexpr int CHUNK = 4;                               // of them joined at a time, one a warp
  static constexpr int PART = ACC * 128 + 2 * COLS;             // floats of a unit's part
  static constexpr int RED = NW * CHUNK * 512;
  static constexpr int CTAS = ctas_of(HD, BITS);
  static constexpr int ROOM = 227 * 1024 / CTAS - RED - 3072;
  static constexpr int STAGES = ROOM / TILE > 8 ? 8 : ROOM / TILE;
  static constexpr int SMEM = STAGES * TILE + RED;
  static_assert(STAGES >= 2, "a ring needs two stages");
  static_assert(CTAS * kSMs <= kCounters, "a counter a CTA");
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
// the same with the low parts in columns 4 .. 7, which repeat columns 0 .. 3
__device__ __forceinline__ uint32_t split_columns(float w0, float w1, bool low) {
  const uint32_t h = pack2(w0, w1), l = pack2(w0 - bf16_lo(h), w1 - bf16_hi(h));
  return transpose8x8(low ? l : h);
}

// (x & mask) | bits as the one instruction that it is (written plainly it became two, a third of a step's instructions),
// and (~x & mask) | bits
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
  return r;
}
__device__ __forceinline__ uint32_t nand_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xae;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
  return r;
}

// two codes of a word (bits 4 i and 4 i + 16) as bf16 128 + c
__device__ __forceinline__ uint32_t codes128(uint32_t w, int i) { return and_or(w >> (4 * i), 0x000f000fu, 0x43004300u); }
// the same as bf16 16 + c (the code in the upper four bits of the mantissa), and as c - 31 = -(16 + (15 - c))
__device__ __forceinline__ uint32_t codes16(uint32_t w, int i) {
  return and_or(i == 0 ? w << 3 : w >> (4 * i - 3), 0x00780078u, 0x41804180u);
}
__device__ __forceinline__ uint32_t codes31(uint32_t w, int i) {
  return nand_or(i == 0 ? w << 3 : w >> (4 * i - 3), 0x00780078u, 0xc180c180u);
}

// The line: units in the order (sequence, key head, column tile), each kPad
// places for what a unit costs beside its tiles (queries, joining, output:
// about that many tiles' time), then its token tiles.  1, 2, 3, 4 places: 64
// sequences of up to 16384 take 145, 138, 139, 140 us, 8 of up to 4096 with 4 new
// rows 34.8, 34.1, 35.5, 36.4: in these two 1 is too few, and 2 to 4 are within 1 and
// 7 % of each other.
constexpr int kPad = 2;

template <int TS, int NC>
struct Line {
  const AttnParams *a;
  const PagedView *c;
  int s, h, ct, n_ct, rows, first, len;   // the current unit
  int tiles;                              // its tiles
  int64_t at;                             // its first place

  // false where something of it had to be left out
  __device__ __forceinline__ bool load(int seq, int &r, int &f, int &l) const {
    f = a->q_off ? a->q_off[seq] : seq;
    r = a->q_off ? a->q_off[seq + 1] - f : 1;
    l = a->kv_len[seq];
    const int most = c->max_pages * c->page;
    const bool inside = f >= 0 && r >= 0 && f <= a->T - r, fits = l >= 0 && l <= most;
    if (!inside) r = 0;   // rows outside q: none
    l = min(max(l, 0), most);
    return inside && fits;
  }
  __device__ __forceinline__ int columns(int r) const { return (r * a->group + NC - 1) / NC; }
  // token tiles up to the last key that a column tile's last row sees
  __device__ __forceinline__ int unit_tiles(int r, int l, int t) const {
    const int last = min(r * a->group, (t + 1) * NC) - 1;
    const int k = l - r + last / a->group + 1;
    return k <= TS ? 1 : (k + TS - 1) / TS;   // a unit without keys still has its output to write
  }
  __device__ __forceinline__ int64_t head_places(int r, int l) const {
    int64_t n = 0;
    for (int t = 0, e = columns(r); t < e; t++) n += kPad + unit_tiles(r, l, t);
    return n;
  }
  // Cuts the line into pieces for `ctas` CTAs and goes to the first unit of
  // piece `me`: [w0, w1), false where there are fewer pieces.
  __device__ bool cut(int ctas, int me, int lane, int64_t &total, int &pieces, int64_t &w0, int64_t &w1) {
    int r = 0, f = 0, l = 0;
    if (lane < c->n_seq) load(lane, r, f, l);
    const int64_t n0 = r ? head_places(r, l) * c->kv_heads : 0;   // sequences 0 .. 31 stay in registers
    total = n0;
    for (int i = lane + 32; i < c->n_seq; i += 32) {
      int r1, f1, l1;
      load(i, r1, f1, l1);
      total += head_places(r1, l1) * c->kv_heads;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    pieces = (int)min((int64_t)ctas, total);   // every piece holds a place
    if (me >= pieces) return false;
    w0 = total * me / pieces;
    w1 = total * (me + 1) / pieces;
    at = 0;
    int64_t n = n0;
    for (int base = 0;; base += 32) {
      if (base) {
        r = 0;
        if (base + lane < c->n_seq) load(base + lane, r, f, l);
        n = r ? head_places(r, l) * c->kv_heads : 0;
      }
      int64_t up = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, at + up > w0);
      if (past) {
        const int hit = __ffs(past) - 1;
        s = base + hit;
        at += __shfl_sync(0xffffffffu, up - n, hit);
        rows = __shfl_sync(0xffffffffu, r, hit);
        first = __shfl_sync(0xffffffffu, f, hit);
        len = __shfl_sync(0xffffffffu, l, hit);
        break;
      }
      at += __shfl_sync(0xffffffffu, up, 31);
    }
    n_ct = columns(rows);
    const int64_t per = head_places(rows, len);
    h = (int)((w0 - at) / per);
    at += h * per;
    ct = 0;
    for (;;) {
      tiles = unit_tiles(rows, len, ct);
      if (w0 < at + kPad + tiles) break;
      at += kPad + tiles;
      ct++;
    }
    return true;
  }
  __device__ __forceinline__ void next() {
    at += kPad + tiles;
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
  // the piece's tiles of the current unit: [t0, t1), empty where it ends inside the unit's first places
  __device__ __forceinline__ void span(int64_t w0, int64_t w1, int &t0, int &t1) const {
    t0 = (int)max(w0 - at - kPad, (int64_t)0);
    t1 = (int)min(w1 - at - kPad, (int64_t)tiles);
  }
};

// Waits for a free stage: the copies' warp has time, and a busy wait would take issue slots from the products.
__device__ __forceinline__ bool wait_free(uint64_t *bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 20); i++) {
    if (mbar_try_wait(bar, parity)) return true;
    __nanosleep(400);
  }
  atomicOr(&g_paged_status, SM100_DECODE_ERR_STALL);
  return false;
}

template <int HD, int BITS, int COLS>
__global__ void __launch_bounds__(Shape<HD, BITS, COLS>::NW * 32 + 32, Shape<HD, BITS, COLS>::CTAS)
    paged_attn_kernel(const __grid_constant__ PagedView c, const __grid_constant__ AttnParams a) {
  using S = Shape<HD, BITS, COLS>;
  constexpr int NW = S::NW, KS = S::KS, TS = S::TS, STAGES = S::STAGES, GR = S::GR, ROW = S::ROW, MARKS = S::MARKS;
  constexpr bool DUAL = S::DUAL;
  extern __shared__ __align__(128) uint8_t smem[];
  float4 *red = reinterpret_cast<float4 *>(smem + STAGES * S::TILE);
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ uint16_t valid[STAGES][TS / 16];
  __shared__ float wm[NW][COLS], wl[NW][COLS], um[COLS], ul[COLS];
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
  Line<TS, COLS> line;
  line.a = &a;
  line.c = &c;
  const int me = blockIdx.x;
  int64_t total, w0, w1;
  int G, t0, t1;
  const auto tell_bad_sequences = [&] {
    for (int s = lane; s < c.n_seq; s += 32) {
      int r, f, l;
      if (!line.load(s, r, f, l)) atomicOr(&g_paged_status, SM100_DECODE_ERR_ARG);
    }
  };
  if (!line.cut(gridDim.x, me, lane, total, G, w0, w1)) {
    if (me == 0 && warp == NW) tell_bad_sequences();   // no rows at all
    return;
  }
  uint32_t it = 0;   // tiles through the ring

  if (warp == NW) {
    // ---- the copies: a lane takes one of a page's areas (keys, their marks, values, their marks)
    constexpr int AREAS = BITS == 4 ? 4 : 2;
    const int area = lane % AREAS, in_tile = lane / AREAS, page = c.page;
    const bool is_v = area >= AREAS / 2, is_marks = BITS == 4 && (area & 1);
    const uint32_t bytes = page * (is_marks ? MARKS : ROW);
    const uint32_t from = (is_v ? c.block / 2 : 0) + (is_marks ? page * ROW : 0);
    uint8_t *to = smem + (is_v ? S::V : 0) + (is_marks ? TS * ROW : 0) + in_tile * bytes;
    const int per = TS >> c.page_log2;            // pages of a tile
    const uint64_t pol = policy_evict_first();
    bool ok_ring = true;
    for (;;) {
      line.span(w0, w1, t0, t1);
      for (int t = t0; t < t1 && ok_ring; t++, it++) {
        const int st = it % STAGES;
        const int slot = t * per + in_tile, key = slot << c.page_log2;
        int id = -1;
        const bool want = in_tile < per && key < line.len;
        if (want) id = c.table[(int64_t)line.s * c.max_pages + slot];
        const bool ok = want && (unsigned)id < (unsigned)c.n_pages;
        if (want && !ok) atomicOr(&g_paged_status, SM100_DECODE_ERR_ARG);
        const uint32_t oks = __ballot_sync(0xffffffffu, ok);
        if (it >= STAGES && !wait_free(&empty[st], (it / STAGES - 1) & 1)) {
          ok_ring = false;
          break;
        }
        if (lane < TS / 16) {
          const int base = t * TS + 16 * lane, n = min(max(line.len - base, 0), 16);
          valid[st][lane] = oks >> (((16 * lane) >> c.page_log2) * AREAS) & 1 ? (uint16_t)((1u << n) - 1) : 0;
        }
        __syncwarp();
        if (lane == 0) mbar_expect_tx(&full[st], __popc(oks) / AREAS * c.block);
        __syncwarp();
        if (ok)
          bulk_g2s_hint(to + st * S::TILE, c.pool + ((int64_t)id * c.kv_heads + line.h) * c.block + from, bytes, &full[st], pol);
      }
      if (!ok_ring || line.at + kPad + line.tiles >= w1) break;
      line.next();
    }
    if (me == 0) tell_bad_sequences();
    return;
  }

  // ---- the products
  const int g = lane >> 2, cq = lane & 3;
  const auto column = [](int col) { return DUAL ? col & 3 : col; };   // the query column of a product's column
  // this thread's places in a tile: tokens g, g + 8 of the keys; 2 cq, 2 cq + 1 and 8 on of the values
  const uint8_t *kp = smem + (16 * KS * warp + g) * ROW + (BITS == 4 ? cq * 8 : cq * 16);
  const uint8_t *vp = smem + S::V + (16 * KS * warp + 2 * cq) * ROW + (BITS == 4 ? g * 4 : g * 16);
  const uint8_t *mp = smem + TS * ROW + (16 * KS * warp + g) * MARKS;   // marks of tokens g, g + 8 (values': V on)
  bool stalled = false;
  for (;; line.next()) {
    line.span(w0, w1, t0, t1);
    if (t0 >= t1) break;   // the piece ends before the unit's first tile
    const int n_cols = min(COLS, line.rows * a.group - line.ct * COLS);
    // Q^T fragments: column g of each 8, this lane's dimensions
    uint32_t qf[HD / 8];
    float qs[GR][2];   // 4 bits: sum of a column's queries over a group (columns 2 cq, 2 cq + 1)
    const int col = column(g), at = line.ct * COLS + col;
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
        qf[4 * i] = __byte_perm(v[i].x, v[i].z, 0x5410);
        qf[4 * i + 1] = __byte_perm(v[i].x, v[i].z, 0x7632);
        qf[4 * i + 2] = __byte_perm(v[i].y, v[i].w, 0x5410);
        qf[4 * i + 3] = __byte_perm(v[i].y, v[i].w, 0x7632);
      } else {
        qf[4 * i] = v[i].x, qf[4 * i + 1] = v[i].y, qf[4 * i + 2] = v[i].z, qf[4 * i + 3] = v[i].w;
      }
    }
    if constexpr (BITS == 4) {
#pragma unroll
      for (int gr = 0; gr < GR; gr++) {
        float s = 0.0f;
#pragma unroll
        for (int i = 8 * gr; i < 8 * gr + 8; i++) s += bf16_lo(qf[i]) + bf16_hi(qf[i]);
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        qs[gr][0] = __shfl_sync(0xffffffffu, s, 8 * cq);
        qs[gr][1] = __shfl_sync(0xffffffffu, s, 8 * cq + 4);
      }
    }
    // keys that this thread's columns see; the smallest of the unit's columns
    int lim[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int col = column(2 * cq + e), at = line.ct * COLS + col;
      lim[e] = col < n_cols ? line.len - line.rows + at / a.group + 1 : 0;
    }
    const int row0 = line.ct * COLS / a.group, row1 = (line.ct * COLS + n_cols - 1) / a.group;
    const int lim_min = line.len - line.rows + row0 + 1;
    float o[GR * 4][4], l[2], m[2], z[GR][2];
#pragma unroll
    for (int i = 0; i < GR * 4; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[i][e] = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      l[e] = 0.0f, m[e] = -INFINITY;
#pragma unroll
      for (int gr = 0; gr < GR; gr++) z[gr][e] = 0.0f;
    }

    for (int t = t0; t < t1; t++, it++) {
      const int st = it % STAGES;
      if (!stalled) stalled = !mbar_wait(&full[st], (it / STAGES) & 1, &g_paged_status, false);
      uint32_t bits[KS];
      uint32_t any_bits = 0;
#pragma unroll
      for (int x = 0; x < KS; x++) any_bits |= bits[x] = stalled ? 0 : valid[st][KS * warp + x];
      if (any_bits != 0) {
        const int in_ring = st * S::TILE;
        const uint8_t *kt = kp + in_ring, *vt = vp + in_ring, *mt = mp + in_ring;
        const int key0 = t * TS + 16 * KS * warp;
        float sc[KS][4];
#pragma unroll
        for (int x = 0; x < KS; x++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[x][e] = 0.0f;
        if constexpr (BITS == 4) {
#pragma unroll
          for (int gr = 0; gr < GR; gr++)
#pragma unroll
            for (int x = 0; x < KS; x++) {
              const uint2 u0 = *reinterpret_cast<const uint2 *>(kt + x * 16 * ROW + gr * 32);
              const uint2 u8 = *reinterpret_cast<const uint2 *>(kt + x * 16 * ROW + 8 * ROW + gr * 32);
              const uint32_t m0 = *reinterpret_cast<const uint32_t *>(mt + x * 16 * MARKS + gr * 4);
              const uint32_t m8 = *reinterpret_cast<const uint32_t *>(mt + x * 16 * MARKS + 8 * MARKS + gr * 4);
              float acc[4];
#pragma unroll
              for (int e = 0; e < 4; e++) acc[e] = 0.0f;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const uint32_t x0 = i < 2 ? u0.x : u0.y, x8 = i < 2 ? u8.x : u8.y;
                const int j = 2 * (i & 1);
                const uint32_t af[4] = {codes128(x0, j), codes128(x8, j), codes128(x0, j + 1), codes128(x8, j + 1)};
                mma_bf16(acc, af, qf[8 * gr + 2 * i], qf[8 * gr + 2 * i + 1]);
              }
              const float s0 = bf16_lo(m0), s8 = bf16_lo(m8);
              const float b0 = fmaf(-128.0f, s0, bf16_hi(m0)), b8 = fmaf(-128.0f, s8, bf16_hi(m8));
#pragma unroll
              for (int e = 0; e < 2; e++) {
                sc[x][e] = fmaf(s0, acc[e], fmaf(b0, qs[gr][e], sc[x][e]));
                sc[x][2 + e] = fmaf(s8, acc[2 + e], fmaf(b8, qs[gr][e], sc[x][2 + e]));
              }
            }
        } else {
#pragma unroll
          for (int i = 0; i < HD / 32; i++)
#pragma unroll
            for (int x = 0; x < KS; x++) {
              const uint4 x0 = *reinterpret_cast<const uint4 *>(kt + x * 16 * ROW + i * 64);
              const uint4 x8 = *reinterpret_cast<const uint4 *>(kt + x * 16 * ROW + 8 * ROW + i * 64);
              const uint32_t a0[4] = {x0.x, x8.x, x0.y, x8.y}, a1[4] = {x0.z, x8.z, x0.w, x8.w};
              mma_bf16(sc[x], a0, qf[4 * i], qf[4 * i + 1]);
              mma_bf16(sc[x], a1, qf[4 * i + 2], qf[4 * i + 3]);
            }
        }
        // tokens that a column does not see, or that are not there
        bool edge = key0 + 16 * KS > lim_min;
#pragma unroll
        for (int x = 0; x < KS; x++) edge |= bits[x] != 0xffffu;
        if (edge) {
#pragma unroll
          for (int x = 0; x < KS; x++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int r = e < 2 ? g : g + 8;
              if (!(bits[x] >> r & 1) || key0 + 16 * x + r >= lim[e & 1]) sc[x][e] = -INFINITY;
            }
        }
        // the running maximum moves only where a column grows past it by 2^8 (a weight of up to 2^8 costs an f32 sum
        // nothing): most tiles then skip the reduction and the rescaling
        float top[2];
        bool grows = false;
#pragma unroll
        for (int e = 0; e < 2; e++) {
          top[e] = fmaxf(sc[0][e], sc[0][2 + e]);
#pragma unroll
          for (int x = 1; x < KS; x++) top[e] = fmaxf(top[e], fmaxf(sc[x][e], sc[x][2 + e]));
          grows |= top[e] * a.scale_log2 > m[e] + 8.0f;
        }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float v = fmaxf(top[e] * a.scale_log2, m[e]);
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, y));
            const float f = v == -INFINITY ? 1.0f : ex2(m[e] - v);
            m[e] = v;
            l[e] *= f;
#pragma unroll
            for (int gr = 0; gr < GR; gr++) z[gr][e] *= f;
#pragma unroll
            for (int i = 0; i < GR * 4; i++) o[i][e] *= f, o[i][2 + e] *= f;
          }
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float mm = m[e] == -INFINITY ? 0.0f : m[e];
#pragma unroll
          for (int x = 0; x < KS; x++) {
            sc[x][e] = ex2(fmaf(sc[x][e], a.scale_log2, -mm));
            sc[x][2 + e] = ex2(fmaf(sc[x][2 + e], a.scale_log2, -mm));
            l[e] += sc[x][e] + sc[x][2 + e];
          }
        }
        if constexpr (BITS == 4) {
#pragma unroll
          for (int gr = 0; gr < GR; gr++)
#pragma unroll
            for (int x = 0; x < KS; x++) {
              const uint8_t *vc = vt + x * 16 * ROW + gr * 32;
              const uint32_t m0 = *reinterpret_cast<const uint32_t *>(mt + S::V + x * 16 * MARKS + gr * 4);
              const uint32_t m8 = *reinterpret_cast<const uint32_t *>(mt + S::V + x * 16 * MARKS + 8 * MARKS + gr * 4);
              const uint32_t wa = *reinterpret_cast<const uint32_t *>(vc);
              const uint32_t wb = *reinterpret_cast<const uint32_t *>(vc + ROW);
              const uint32_t wc = *reinterpret_cast<const uint32_t *>(vc + 8 * ROW);
              const uint32_t wd = *reinterpret_cast<const uint32_t *>(vc + 9 * ROW);
              const float s0 = bf16_lo(m0), s8 = bf16_lo(m8);
              const float b0 = fmaf(-16.0f, s0, bf16_hi(m0)), b8 = fmaf(31.0f, s8, bf16_hi(m8));
              uint32_t p0, p8, r0, r8;
              float w[4];
              if (!edge) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  w[e] = sc[x][e] * s0, w[2 + e] = sc[x][2 + e] * s8;
                  z[gr][e] = fmaf(sc[x][e], b0, fmaf(sc[x][2 + e], b8, z[gr][e]));
                }
              } else {   // a weight of zero leaves out whatever the token holds
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  const bool k0 = sc[x][e] != 0.0f, k8 = sc[x][2 + e] != 0.0f;
                  w[e] = k0 ? sc[x][e] * s0 : 0.0f, w[2 + e] = k8 ? sc[x][2 + e] * s8 : 0.0f;
                  if (k0) z[gr][e] += sc[x][e] * b0;
                  if (k8) z[gr][e] += sc[x][2 + e] * b8;
                }
              }
              if constexpr (DUAL) {
                p0 = split_columns(w[0], w[1], cq >= 2);
                p8 = split_columns(w[2], w[3], cq >= 2);
              } else {
                split_weights(w[0], w[1], p0, r0);
                split_weights(w[2], w[3], p8, r8);
              }
              const uint32_t lo[2] = {__byte_perm(wa, wb, 0x5410), __byte_perm(wa, wb, 0x7632)};
              const uint32_t hi[2] = {__byte_perm(wc, wd, 0x5410), __byte_perm(wc, wd, 0x7632)};
#pragma unroll
              for (int j = 0; j < 4; j++) {   // dimensions 8 g + 2 j, 8 g + 2 j + 1 of the group
                const int i = 2 * (j & 1);
                const uint32_t af[4] = {codes16(lo[j >> 1], i), codes16(lo[j >> 1], i + 1), codes31(hi[j >> 1], i),
                                        codes31(hi[j >> 1], i + 1)};
                mma_bf16(o[4 * gr + j], af, p0, p8);
                if constexpr (!DUAL) mma_bf16(o[4 * gr + j], af, r0, r8);
              }
            }
        } else {
          const int k0 = 2 * cq, tk[4] = {k0, k0 + 1, k0 + 8, k0 + 9};
#pragma unroll
          for (int x = 0; x < KS; x++) {
            const uint8_t *vc = vt + x * 16 * ROW;
            uint32_t p0, p8, r0, r8;
            split_weights(sc[x][0], sc[x][1], p0, r0);
            split_weights(sc[x][2], sc[x][3], p8, r8);
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
              uint4 v[4];
#pragma unroll
              for (int k = 0; k < 4; k++) v[k] = *reinterpret_cast<const uint4 *>(vc + gr * 128 + (k >> 1) * 8 * ROW + (k & 1) * ROW);
              if (!edge) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  const uint32_t wa = (&v[0].x)[j], wb = (&v[1].x)[j], wc = (&v[2].x)[j], wd = (&v[3].x)[j];
                  const uint32_t af[4] = {__byte_perm(wa, wb, 0x5410), __byte_perm(wa, wb, 0x7632),
                                          __byte_perm(wc, wd, 0x5410), __byte_perm(wc, wd, 0x7632)};
                  mma_bf16(o[4 * gr + j], af, p0, p8);
                  mma_bf16(o[4 * gr + j], af, r0, r8);
                }
              } else {
                // row by row: a token that a row does not see is zeros to it, and another row's product, where that
                // token may hold an infinity or a NaN, does not enter its columns
                for (int r = row0; r <= row1; r++) {
                  const int seen = line.len - line.rows + r + 1;
                  uint32_t keep[4];
#pragma unroll
                  for (int k = 0; k < 4; k++)
                    keep[k] = (bits[x] >> tk[k] & 1) && key0 + 16 * x + tk[k] < seen ? 0xffffffffu : 0u;
#pragma unroll
                  for (int j = 0; j < 4; j++) {
                    const uint32_t wa = (&v[0].x)[j] & keep[0], wb = (&v[1].x)[j] & keep[1];
                    const uint32_t wc = (&v[2].x)[j] & keep[2], wd = (&v[3].x)[j] & keep[3];
                    const uint32_t af[4] = {__byte_perm(wa, wb, 0x5410), __byte_perm(wa, wb, 0x7632),
                                            __byte_perm(wc, wd, 0x5410), __byte_perm(wc, wd, 0x7632)};
                    float tmp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_bf16(tmp, af, p0, p8);
                    mma_bf16(tmp, af, r0, r8);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                      if (lim[e & 1] == seen) o[4 * gr + j][e] += tmp[e];
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

    // ---- the warps' parts of the unit joined.  A maximum of -inf: no token that counts, a sum of 0, or none but scores of
    // NaN (which a maximum passes over), a sum of NaN: the sum then stands for the part's weight
    const bool mine = !DUAL || cq < 2;   // this thread's columns are query columns
#pragma unroll
    for (int e = 0; e < 2; e++) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
        if constexpr (BITS == 4) {
#pragma unroll
          for (int gr = 0; gr < GR; gr++) z[gr][e] += __shfl_xor_sync(0xffffffffu, z[gr][e], x);
        }
      }
      if (g == 0 && mine) wm[warp][2 * cq + e] = m[e], wl[warp][2 * cq + e] = l[e];
    }
    const auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(NW * 32) : "memory"); };
    sync();
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int col = column(2 * cq + e);
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NW; i++) top = fmaxf(top, wm[i][col]);
#pragma unroll
      for (int i = 0; i < NW; i++) sum += wm[i][col] == -INFINITY ? wl[i][col] : wl[i][col] * ex2(wm[i][col] - top);
      f[e] = m[e] == -INFINITY ? l[e] : ex2(m[e] - top);
      if (warp == 0 && g == 0 && mine) um[col] = top, ul[col] = sum;
    }
    // where the piece ends inside the unit, or began inside it: a part
    const bool whole = t0 == 0 && t1 == line.tiles;
    float *part = a.parts + ((int64_t)me * 2 + (t0 == 0)) * S::PART;
    // an accumulator tile's values: dimensions d, d + 1 of columns 2 cq, 2 cq + 1
    const auto put = [&](int i, float4 v) {
      const int d = (i >> 2) * 64 + 8 * g + 2 * (i & 3);
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int col = 2 * cq + e, at = line.ct * COLS + col;
        if (!mine || col >= n_cols) continue;
        const float inv = ul[col] > 0.0f ? 1.0f / ul[col] : ul[col] == 0.0f ? 0.0f : ul[col];
        *reinterpret_cast<uint32_t *>(a.out + ((int64_t)(line.first + at / a.group) * a.heads + line.h * a.group + at % a.group) * HD + d) =
            e ? pack2(v.y * inv, v.w * inv) : pack2(v.x * inv, v.z * inv);
      }
    };
    const bool used = mine && 2 * cq < n_cols;   // a lane without query columns has nothing to join (its low parts are added)
    for (bool last = whole;; last = true) {
#pragma unroll
      for (int ch = 0; ch < S::ACC / S::CHUNK; ch++) {
#pragma unroll
        for (int k = 0; k < S::CHUNK; k++) {
          const int i = ch * S::CHUNK + k;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            v[e] = o[i][e];
            if constexpr (DUAL) v[e] += __shfl_xor_sync(0xffffffffu, v[e], 2);
            if constexpr (BITS == 4) v[e] += z[i >> 2][e & 1];
            v[e] = f[e & 1] == 0.0f ? 0.0f : v[e] * f[e & 1];
          }
          if (used) red[(warp * S::CHUNK + k) * 32 + lane] = make_float4(v[0], v[1], v[2], v[3]);
        }
        sync();
        if (used) {
          const int at = ch * S::CHUNK + warp;   // a warp's tile, over the warps
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int x = 0; x < NW; x++) {
            const float4 u = red[(x * S::CHUNK + warp) * 32 + lane];
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
          }
          if (last) put(at, v);
          else __stcg(reinterpret_cast<float4 *>(part) + at * 32 + lane, v);
        }
        sync();
      }
      if (last) break;
      // a part: the last of the unit's CTAs to come joins all of them, a warp every fourth part
      if (tid < COLS) {
        __stcg(part + S::ACC * 128 + tid, um[tid]);
        __stcg(part + S::ACC * 128 + COLS + tid, ul[tid]);
      }
      // the CTAs that share the unit, by the places of its first and last tile
      const int64_t u0 = line.at + kPad, u1 = u0 + line.tiles - 1;
      const int c0 = (int)(((u0 + 1) * G - 1) / total), c1 = (int)(((u1 + 1) * G - 1) / total);
      __threadfence();
      sync();
      if (tid == 0) arrived = atomicAdd(&a.counters[c0], 1u);
      sync();
      if (arrived != (uint32_t)(c1 - c0)) break;
      __threadfence();
      if (tid == 0) a.counters[c0] = 0;
      const auto part_of = [&](int x) { return a.parts + ((int64_t)x * 2 + (x == c0)) * S::PART; };
      // a column's maximum and sum over the parts, a warp to a column; its weights for kBatch parts at a time
      constexpr int kBatch = S::RED / 4 / COLS;
      float *weights = reinterpret_cast<float *>(red);
      for (int col = warp; col < COLS; col += NW) {
        float top = -INFINITY, sum = 0.0f;
        for (int x = c0 + lane; x <= c1; x += 32) {
          const float *p = part_of(x) + S::ACC * 128 + col;
          const float pm = __ldcg(p), pl = __ldcg(p + COLS);
          if (pm == -INFINITY) {
            sum += pl;
            continue;
          }
          const float v = fmaxf(top, pm);
          sum = sum * ex2(top - v) + pl * ex2(pm - v);
          top = v;
        }
        const float all = warp_max(top);
        sum = warp_sum(top == -INFINITY ? sum : sum * ex2(top - all));
        if (lane == 0) um[col] = all, ul[col] = sum;
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        f[e] = 1.0f;
#pragma unroll
        for (int gr = 0; gr < GR; gr++) z[gr][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < GR * 4; i++) o[i][e] = o[i][2 + e] = 0.0f;
      }
      for (int x0 = c0; x0 <= c1; x0 += kBatch) {
        const int n = min(kBatch, c1 - x0 + 1);
        sync();
        for (int i = tid; i < n * COLS; i += NW * 32) {
          const float pm = __ldcg(part_of(x0 + i / COLS) + S::ACC * 128 + i % COLS);
          weights[i] = pm == -INFINITY ? 0.0f : ex2(pm - um[i % COLS]);   // (a sum of NaN is in the unit's)
        }
        sync();
        // a warp's parts, UN of them under way at a time; with 4 columns the idle half of the lanes takes every other one
        // (the joining adds its columns to the first half's)
        constexpr int UN = S::ACC <= 8 ? 2 : 1, SIDES = DUAL ? 2 : 1;
        const int side = DUAL ? cq >> 1 : 0;
        if (DUAL || used)
          for (int x = warp + NW * side; x < n; x += NW * SIDES * UN) {
            float4 u[UN][S::ACC];
#pragma unroll
            for (int k = 0; k < UN; k++) {
              const int y = x + k * NW * SIDES;
              const float4 *p = reinterpret_cast<const float4 *>(part_of(x0 + y)) + (DUAL ? lane & ~2 : lane);
#pragma unroll
              for (int i = 0; i < S::ACC; i++) u[k][i] = y < n ? __ldcg(p + i * 32) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int k = 0; k < UN; k++) {
              const int y = min(x + k * NW * SIDES, n - 1);
#pragma unroll
              for (int j = 0; j < S::ACC; j++) {
                const int col = column(2 * cq);
                const float f0 = weights[y * COLS + col], f1 = weights[y * COLS + col + 1];
                if (f0 != 0.0f) o[j][0] += u[k][j].x * f0, o[j][2] += u[k][j].z * f0;
                if (f1 != 0.0f) o[j][1] += u[k][j].y * f1, o[j][3] += u[k][j].w * f1;
              }
            }
          }
      }
      sync();
    }
    if (line.at + kPad + line.tiles >= w1) break;
  }
  if (stalled && warp == 0)   // a wait gave up: the copies still under way may not outlive the CTA's shared memory
    for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; i++)
      mbar_wait(&full[i % STAGES], (i / STAGES) & 1, &g_paged_status, false);
}

template <int HD, int BITS, int COLS>
int launch(const PagedView &v, AttnParams &p, const Sm100PagedAttnArgs *a, cudaStream_t st) {
  using S = Shape<HD, BITS, COLS>;
  static int grid[64];   // CTAs that one device holds at once, by ordinal
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev >= 64) return sm100_set_error(SM100_ERR_CUDA, "paged_attention: device %d: %s", dev, cudaGetErrorString(e));
  const auto kernel = paged_attn_kernel<HD, BITS, COLS>;
  if (!grid[dev]) {
    int sms = 0, per = 0;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM)) != cudaSuccess ||
        (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess ||
        (e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, S::NW * 32 + 32, S::SMEM)) != cudaSuccess)
      return sm100_set_error(SM100_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
    if (per < 1) return sm100_set_error(SM100_ERR_UNSUPPORTED, "paged_attention: no room for %d bytes of shared memory", S::SMEM);
    const int most = kSMs * S::CTAS;   // what the scratch holds parts for
    grid[dev] = sms * per < most ? sms * per : most;
  }
  p.counters = static_cast<uint32_t *>(a->ws);
  p.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(a->ws) + kCounters * 4);
  e = launch_pdl(kernel, dim3(grid[dev]), dim3(S::NW * 32 + 32), S::SMEM, st, v, p);
  if (e != cudaSuccess) return sm100_set_error(SM100_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
  return launch_status("paged_attention");
}

// Query columns of a unit
int columns_of(int bits, int64_t cols) { return cols > 4 || bits == 16 ? 8 : 4; }

template <int HD, int BITS>
int launch_columns(const PagedView &v, AttnParams &p, const Sm100PagedAttnArgs *a, cudaStream_t st) {
  if constexpr (BITS == 4) {
    if (columns_of(BITS, (int64_t)a->max_rows * p.group) == 4) return launch<HD, BITS, 4>(v, p, a, st);
  }
  return launch<HD, BITS, 8>(v, p, a, st);
}

}  // namespace

extern "C" uint64_t sm100_paged_attention_ws_bytes(const Sm100PagedCache *c, int32_t heads, int32_t max_rows) {
  PagedView v;
  if (sm100_paged_view(c, "paged_attention_ws_bytes", &v) || heads < 1 || heads % c->kv_heads || max_rows < 1) return 0;
  const uint64_t cols = columns_of(c->bits, (int64_t)max_rows * (heads / c->kv_heads));
  return kCounters * 4 + (uint64_t)kSMs * ctas_of(c->head_dim, c->bits) * 2 * (8 * c->head_dim + 2 * cols) * 4;
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
  if (!(a->scale >= 0.0f && a->scale <= 2e38f))   // times log2(e) it is finite
    return sm100_set_error(SM100_ERR_ARG, "paged_attention: scale %g (0 to 2e38)", (double)a->scale);
  if ((int64_t)a->T * a->heads / c->kv_heads > INT32_MAX)
    return sm100_set_error(SM100_ERR_ARG, "paged_attention: %d rows in one call", a->T);
  AttnParams p{static_cast<const __nv_bfloat16 *>(a->q), a->kv_len, a->q_off, static_cast<__nv_bfloat16 *>(a->out),
               nullptr, nullptr, ld, a->T, a->heads, a->heads / c->kv_heads,
               // a hidden token's score is -inf before it is scaled, and -inf * 0 is NaN: a scale of 0 goes in as the smallest
               // normal number, with which scores below 2^100 come out as 0 to f32's last bit
               fmaxf(a->scale * 1.4426950408889634f, FLT_MIN)};
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
