// Attention of a chunk of new tokens over the paged K/V cache (sequences with more than 32 query rows per kv head and head set), on
// tcgen05, TMEM and TMA.
//
// An item is 256 query rows of one kv head in two tiles of 128: `hp` heads that share it x 256 / hp tokens, the first half of the
// tokens in one tile and the second in the other. The key tiles some row sees are walked 128 keys at a time; S = Q K^T and O += P V
// on the tensor cores with P read from tensor memory, the softmax thread per row in fp32 with P rounded to bf16 for the product. A
// row's reference maximum moves (and O is scaled) only when its maximum has outgrown it by more than 2^24.
//   D 256 (paged_pair_kernel): a CTA pair, one tile of rows each (O takes half of tensor memory). The pair is there for K and V: 128
//       rows alone would need 128 keys from L2 every 2 048 cycles, 64 bytes per cycle and SM, more than L2 delivers. Two S buffers; two
//       groups of four softmax warps, each half the keys of every row. 2 048 tokens over 18 432 (16 / 8 heads of 256): 508 to 558 us, about 2 970
//       cycles a tile where the products take 2 048; the tensor pipe is 61 to 70 % busy, at a clock that the power limit has brought
//       to about 1.6 GHz: 1 037 TFLOP/s of visible pairs.
//   D 128 (paged_two_kernel): one CTA holds both tiles (S and O of each fill tensor memory) and a group of four softmax warps per tile.
//       The exponentials take as long as the products here (128 x 128 at 16 per cycle and SM: 1 024 cycles); with two independent tiles
//       one tile's softmax runs under the other's products and waits, where the pair form left its chain of waits exposed. About
//       4 000 cycles for two tiles (the pair form: 4 870): 2 000 of softmax arithmetic, the rest waits for the products. 1 024 tokens
//       over 8 192 (32 / 16 heads of 128) 150 us; seven chunks of up to 1 501 tokens, window 1 024, 254 us.
// Bound by the chain product - softmax - product; the tensor pipe (4 D flops per row and key) is the floor.
//
// A sequence's work, the (item, key tile) pairs in order, is dealt out in equal contiguous units, one per CTA pair / CTA of the GPU
// (fewer for little work): the causal triangle, ragged tails and few items of many tiles balance by themselves. An item cut by
// a unit's border leaves partial rows (maximum, sum, O in fp32), which the join adds in order. The cut depends on the sequence's own
// lengths only, so its results do not depend on the rest of the call. A front that several sequences share is cut and computed like a
// sequence whose rows see all of it; its items always leave parts, and the join adds the sequences' own splits to them.
#include "paged_attn.cuh"

#include <atomic>

namespace spinf {

static constexpr int CH_KH = 64;
static constexpr float CH_RESCALE = 24.f;  // log2 units: the reference maximum moves when a row's maximum grew by more
static constexpr int CHUNK_THREADS = 384;  // 12 warps (three per scheduler: 168 registers a thread)

template <int D>
struct ChunkSmem {
  static constexpr int SLABS = D / 64;
  static constexpr int Q_BYTES = (D == 256 ? 1 : 2) * SLABS * 128 * 128;   // the CTA's rows of q
  static constexpr int KV = (D == 256 ? CH_KH : PG_TILE) * SLABS * 128;     // one stage: the CTA's share of a tile of K, or of V
  static constexpr int NS = 2;
  static constexpr int SEGS = 8, PLAN = 8;  // segment ring; units planned at a time
  static constexpr int K_OFF = Q_BYTES;
  static constexpr int V_OFF = K_OFF + NS * KV;
  static constexpr int OUT_OFF = V_OFF + NS * KV;   // 2 KB per softmax warp: rows of the output on their way to global memory
  static constexpr int BAR_OFF = OUT_OFF + 8 * 2048;
  static constexpr int XCHG_OFF = BAR_OFF + 512;
  static constexpr int SEG_OFF = XCHG_OFF + 3 * 2 * 128 * 4;
  static constexpr int PLAN_OFF = SEG_OFF + SEGS * 64;
  static constexpr int PRE_OFF = PLAN_OFF + PLAN * 128;
  static constexpr int TOTAL = PRE_OFF + (PG_MAX_SEQS + 2) * 4 + 1024;
  static constexpr int TMEM_COLS = 512;  // D 256: S 2 x 128 columns, O 256; D 128: S of each tile, O of each tile
  static constexpr int O_COL = 256;
};
static_assert(ChunkSmem<256>::TOTAL <= 232448 && ChunkSmem<128>::TOTAL <= 232448, "shared memory of a CTA");

__device__ __forceinline__ void tma_load_5d_pair(void* dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, int c4, uint32_t bar_cluster_addr) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster_addr), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
// an arrival that publishes this CTA's shared-memory writes to the pair's leader
__device__ __forceinline__ void mbar_arrive_cluster_release(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// a segment: consecutive key tiles of one item
struct ChunkSeg {
  int b, row0, nq, base;  // sequence, its first row of q, its rows, the first one's slot
  int g, h0, tok0;        // kv head, first query head, first token
  int ta, tb;             // key tiles (ta < 0: no more segments)
  int lo, hi;             // slots some row of the item sees
  int part;               // partial result (256 rows) to write, or -1: the segment is the whole item
};
static_assert(sizeof(ChunkSeg) <= 64, "slot of the segment ring");

// the walk over a unit's segments, as it is planned
struct ChunkWalk {
  PagedSeq q;
  ChunkCut c;
  int b, it;
  int w, w_end;      // (item, tile) pairs of the unit still to do
  int tt, nt, t0;    // token tile, its key tiles, the first of them
  int w_tt;          // first pair of the token tile
  bool first;

  __device__ __forceinline__ void start(const PagedSeqs& s, const PagedAttnArgs& a, const int* pre, int unit, int* status) {
    b = paged_find(pre, s.B, unit);
    chunk_seq(s, a, b, q, status);
    c = chunk_cut(q, a);
    it = unit;
    const int u = unit - pre[b];
    first = true;
    tt = 0, w_tt = 0;
    ChunkJoin join;
    join.pieces = 0;
    join.b0 = b;
    join.b1 = q.cap != PG_NO_CAP ? s.share[s.B + b] : 0;
    if (c.parts) {
      const int i = u / c.parts, part = u - i * c.parts;
      tt = i / c.per_tt;
      c.tiles(q, a, tt, t0, nt);
      const int item = i - tt * c.per_tt;
      w = item * nt + nt * part / c.parts;  // (pairs counted from the token tile's first)
      w_end = item * nt + nt * (part + 1) / c.parts;
      // parts are the first segments of their units. A front is never whole: its one part is joined with the sequences' own splits
      if (part == 1 || (join.b1 && c.parts == 1)) {
        join.pieces = c.parts;
        join.first = (unit - part) * a.unit_slots;
        join.row0 = q.row0, join.nq = q.nq;
        join.tok0 = tt << c.tok_log2;
        join.h0 = item / a.sets * a.group + (item % a.sets << a.hp_log2);
      }
      a.joins[unit] = join;
      return;
    }
    w = c.begin(u);
    w_end = c.begin(u + 1);
    c.tiles(q, a, 0, t0, nt);
    advance(a);
    const int item = (w - w_tt) / nt, off = w - w_tt - item * nt;
    if (off) {
      if (c.whole) {
        w += nt - off;
      } else if (c.begin(u - 1) <= w - off) {  // the first unit that begins inside this item
        const int w0 = w - off;
        join.pieces = c.unit_of(w0 + nt - 1) - u + 2;
        join.first = (unit - 1) * a.unit_slots + (c.begin(u - 1) < w0 ? 1 : 0);
        join.row0 = q.row0, join.nq = q.nq;
        join.tok0 = tt << c.tok_log2;
        join.h0 = item / a.sets * a.group + (item % a.sets << a.hp_log2);
      }
    }
    a.joins[unit] = join;
  }
  // to the token tile that holds pair w
  __device__ __forceinline__ void advance(const PagedAttnArgs& a) {
#pragma unroll 1
    while (w >= w_tt + nt * c.per_tt && tt + 1 < c.ntt) {
      w_tt += nt * c.per_tt;
      c.tiles(q, a, ++tt, t0, nt);
    }
  }
  __device__ __forceinline__ bool next(const PagedAttnArgs& a, ChunkSeg& g) {
    if (w >= w_end) return false;
    if (!c.parts) advance(a);
    const int item = (w - w_tt) / nt, off = w - w_tt - item * nt;
    const int len = !c.whole && w_end - w < nt - off ? w_end - w : nt - off;
    g.b = b, g.row0 = q.row0, g.nq = q.nq, g.base = q.len - q.nq;
    g.g = item / a.sets;
    g.h0 = g.g * a.group + ((item - g.g * a.sets) << a.hp_log2);
    g.tok0 = tt << c.tok_log2;
    g.ta = t0 + off;
    g.tb = g.ta + len;
    c.slots(q, a, tt, g.lo, g.hi);
    g.part = len == nt && q.cap == PG_NO_CAP ? -1 : it * a.unit_slots + (first ? 0 : 1);  // (one slot: units are parts, of one segment each)
    first = false;
    w += len;
    return true;
  }
};
static_assert(sizeof(ChunkWalk) <= 128, "slot of the unit plan");

// The segments reach the other warps through a ring in shared memory: units are planned several at a time, one per lane, so that none
// of the searches and divisions stands between two segments.
template <class L>
struct SegRing {
  ChunkSeg* slots;
  uint64_t* full;
  uint64_t* empty;
  uint32_t n;
  __device__ __forceinline__ bool next(const WaitCtx& wc, ChunkSeg& g) const {
    if (!mbar_wait(wc, &full[n % L::SEGS], (n / L::SEGS) & 1u, ST_TIMEOUT_FULL)) return false;
    g = *reinterpret_cast<const ChunkSeg*>(reinterpret_cast<const uint8_t*>(slots) + (n % L::SEGS) * 64);
    return g.ta >= 0;
  }
  // one arrival per reading warp; the numbers are in registers from here on
  __device__ __forceinline__ void done() { mbar_arrive(&empty[n++ % L::SEGS]); }
};
// the planning side (one warp): publish() puts the next segment into the ring, at the end the mark that there is none
template <class L>
struct SegPlan {
  uint8_t* plan;   // L::PLAN walks of 128 bytes
  int u, k, total, step;  // next unit to plan for, next walk
  uint32_t n;
  bool ended;
  __device__ __forceinline__ bool publish(const PagedSeqs& s, const PagedAttnArgs& a, const int* pre, const SegRing<L>& ring, const WaitCtx& wc, int* status) {
    if (ended) return true;
    const int lane = threadIdx.x & 31;
    for (;;) {
      if (k == L::PLAN && u < total) {
        __syncwarp();
        const int mine = u + lane * step;
        if (lane < L::PLAN && mine < total) {
          ChunkWalk wk;
          wk.start(s, a, pre, mine, status);
          *reinterpret_cast<ChunkWalk*>(plan + lane * 128) = wk;
        }
        __syncwarp();
        k = 0;
      }
      const bool have = k < L::PLAN && u + k * step < total;
      int put = 0;  // 1: a segment, 2: the walk has none left, 3: the ring does not empty
      if (lane == 0) {
        ChunkSeg g;
        g.ta = -1;
        put = 1;
        if (have) {
          ChunkWalk wk = *reinterpret_cast<const ChunkWalk*>(plan + k * 128);
          put = wk.next(a, g) ? 1 : 2;
          *reinterpret_cast<ChunkWalk*>(plan + k * 128) = wk;
        }
        if (put == 1) {
          if (mbar_wait(wc, &ring.empty[n % L::SEGS], ((n / L::SEGS) & 1u) ^ 1u, ST_TIMEOUT_EMPTY)) {
            *reinterpret_cast<ChunkSeg*>(reinterpret_cast<uint8_t*>(ring.slots) + (n % L::SEGS) * 64) = g;
            mbar_arrive(&ring.full[n % L::SEGS]);
          } else {
            put = 3;
          }
        }
      }
      put = __shfl_sync(0xffffffffu, put, 0);
      if (put == 2) {
        if (++k == L::PLAN) u += L::PLAN * step;
        continue;
      }
      ++n;
      ended = !have;
      return put == 1;
    }
  }
};

// The pages of a segment's boxes in the order they are copied, 32 fetched at a time by the lanes of the producer warp and the next 32
// ahead of use: the copy loop never waits for a table entry.
struct PageRun {
  int cur, nxt, x;       // box
  int j0, nb_log2, rl;   // first slot of box 0; boxes per tile, rows of a box (log2)
  __device__ __forceinline__ int fetch(const PagedSeqs& s, const int32_t* pages, const ChunkSeg& g, int box, int* status) const {
    const int t = g.ta + (box >> nb_log2);
    if (t >= g.tb) return s.n_pages;
    return chunk_page(s, pages, t * PG_TILE + j0 + ((box & ((1 << nb_log2) - 1)) << rl), 1 << rl, g.lo, g.hi, status);
  }
  __device__ __forceinline__ void start(const PagedSeqs& s, const int32_t* pages, const ChunkSeg& g, int first, int boxes_log2, int rows_log2, int lane, int* status) {
    x = 0, j0 = first, nb_log2 = boxes_log2, rl = rows_log2;
    cur = fetch(s, pages, g, lane, status);
    nxt = fetch(s, pages, g, 32 + lane, status);
  }
  __device__ __forceinline__ int get(const PagedSeqs& s, const int32_t* pages, const ChunkSeg& g, int lane, int* status) {
    if (x && (x & 31) == 0) {
      cur = nxt;
      nxt = fetch(s, pages, g, x + 32 + lane, status);
    }
    return __shfl_sync(0xffffffffu, cur, x++ & 31);
  }
};

// O of 128 rows x COLS columns from tensor memory (from column `taddr`, head dimensions from d0 on): divided by the sums and rounded to
// the output, or in fp32 to the segment's partial result. `free_o` is called when the last column is in registers. A warp's 32 rows go
// through 2 KB of shared memory, so that a store instruction covers whole sectors side by side (8 rows x 64 bytes, 4 rows x 128 bytes)
// instead of 16 bytes of 32 rows; where the rows go is worked out once for all columns.
template <int D, int COLS, class Free>
__device__ __forceinline__ void chunk_store(const PagedAttnArgs& a, const ChunkSeg& g, uint32_t taddr, int d0, int tile, int qd, int lane, float inv,
                                            uint8_t* stage, Free free_o) {
  uint4* st = reinterpret_cast<uint4*>(stage);
  if (g.part < 0) {
    const int ql = 7 - a.hp_log2;  // log2 of a head's rows in a tile
    __nv_bfloat16* to[4];          // rows lane / 4, + 8, + 16, + 24 of the warp (null: none of the sequence's)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int rr = qd * 32 + k * 8 + (lane >> 2);
      const int tok = g.tok0 + (tile << ql) + (rr & ((1 << ql) - 1)), head = g.h0 + (rr >> ql);
      to[k] = tok < g.nq ? a.out + static_cast<int64_t>(g.row0 + tok) * a.out_pitch + head * D + d0 + (lane & 3) * 8 : nullptr;
    }
    const int rd = (lane >> 2) * 4 + ((lane & 3) ^ ((lane >> 3) & 3));  // (rows 8 apart swizzle alike)
#pragma unroll 1
    for (int c = 0; c < COLS; c += 32) {
      uint32_t o[32];
      __syncwarp();
      tmem_ld_x32(taddr + c, o);
      tmem_wait_ld();
      if (c + 32 >= COLS) free_o();
#pragma unroll
      for (int x = 0; x < 4; ++x)
        st[lane * 4 + (x ^ ((lane >> 1) & 3))] =
            make_uint4(pack_bf16x2(__uint_as_float(o[8 * x]) * inv, __uint_as_float(o[8 * x + 1]) * inv),
                       pack_bf16x2(__uint_as_float(o[8 * x + 2]) * inv, __uint_as_float(o[8 * x + 3]) * inv),
                       pack_bf16x2(__uint_as_float(o[8 * x + 4]) * inv, __uint_as_float(o[8 * x + 5]) * inv),
                       pack_bf16x2(__uint_as_float(o[8 * x + 6]) * inv, __uint_as_float(o[8 * x + 7]) * inv));
      __syncwarp();
      uint4 w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = st[k * 32 + rd];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (to[k]) *reinterpret_cast<uint4*>(to[k] + c) = w[k];
    }
  } else {
    float* to = a.chunk_o + (static_cast<int64_t>(g.part) * 256 + tile * 128 + qd * 32 + (lane >> 3)) * D + d0 + (lane & 7) * 4;
#pragma unroll 1
    for (int c = 0; c < COLS; c += 32) {
      uint32_t o[32];
      __syncwarp();
      tmem_ld_x32(taddr + c, o);
      tmem_wait_ld();
      if (c + 32 >= COLS) free_o();
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 128 bytes of 16 rows at a time
        if ((lane >> 4) == h) {
#pragma unroll
          for (int x = 0; x < 8; ++x) st[(lane & 15) * 8 + (x ^ (lane & 7))] = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
        }
        __syncwarp();
        uint4 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = st[k * 32 + (lane & ~7) + ((lane & 7) ^ ((k * 4 + (lane >> 3)) & 7))];
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<uint4*>(to + c + (h * 16 + k * 4) * D) = w[k];
        __syncwarp();
      }
    }
  }
}
__device__ __forceinline__ void chunk_store_stats(const PagedAttnArgs& a, const ChunkSeg& g, int tile, int row, int tok, int head, float m, float l) {
  if (tok >= g.nq) return;
  if (g.part >= 0)
    a.chunk_ml[static_cast<int64_t>(g.part) * 256 + tile * 128 + row] = make_float2(m, l);
  else if (a.lse)
    a.lse[static_cast<int64_t>(g.row0 + tok) * a.H + head] = m + log2f(l);
}

// 64 scores of a row from tensor memory, hidden ones (slots outside [lo, hi], jb the first's slot) at -inf where the tile is a boundary
__device__ __forceinline__ void chunk_scores(float (&sc)[64], uint32_t taddr, bool masked, int jb, int lo, int hi) {
  uint32_t v0[32], v1[32];
  tmem_ld_x32(taddr, v0);
  tmem_ld_x32(taddr + 32, v1);
  tmem_wait_ld();
#pragma unroll
  for (int c = 0; c < 32; ++c) sc[c] = __uint_as_float(v0[c]), sc[32 + c] = __uint_as_float(v1[c]);
  if (masked) {
    uint64_t bits = hi < jb ? 0ull : hi - jb >= 63 ? ~0ull : (2ull << (hi - jb)) - 1ull;
    if (lo > jb) bits &= lo - jb > 63 ? 0ull : ~0ull << (lo - jb);
    const uint32_t b_lo = static_cast<uint32_t>(bits), b_hi = static_cast<uint32_t>(bits >> 32);
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      sc[c] = (b_lo & (1u << c)) ? sc[c] : -INFINITY;
      sc[32 + c] = (b_hi & (1u << c)) ? sc[32 + c] : -INFINITY;
    }
  }
}
__device__ __forceinline__ float chunk_max(const float (&sc)[64]) {
  float m[4] = {sc[0], sc[1], sc[2], sc[3]};  // four chains: one is 64 dependent instructions
#pragma unroll
  for (int c = 4; c < 64; ++c) m[c & 3] = fmaxf(m[c & 3], sc[c]);
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// p = 2^(scale s - m), packed to bf16 pairs; returns their sum (unrounded)
__device__ __forceinline__ float chunk_probs(const float (&sc)[64], float scale_log2, float neg_m, uint32_t (&pk)[32]) {
  float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const float p0 = fast_exp2(fmaf(sc[2 * c], scale_log2, neg_m)), p1 = fast_exp2(fmaf(sc[2 * c + 1], scale_log2, neg_m));
    sum0 += p0;
    sum1 += p1;
    pk[c] = pack_bf16x2(p0, p1);
  }
  return sum0 + sum1;
}
__device__ __forceinline__ uint32_t slot_bits(int jb, int lo, int hi) {  // which of the 32 slots from jb on lie in [lo, hi]
  uint32_t bits = hi < jb ? 0u : hi - jb >= 31 ? ~0u : (2u << (hi - jb)) - 1u;
  if (lo > jb) bits &= lo - jb > 31 ? 0u : ~0u << (lo - jb);
  return bits;
}
// P of 64 keys of a row from their scores in tensor memory, and on the way the largest score; sum: of p, unrounded
__device__ __forceinline__ float chunk_half(uint32_t taddr, bool masked, int jb, int lo, int hi, float scale_log2, float neg_m, uint32_t (&pk)[32], float& sum) {
  float m[2] = {-INFINITY, -INFINITY}, s[2] = {0.f, 0.f};
  uint32_t v0[32], v1[32];
  tmem_ld_x32(taddr, v0);
  tmem_ld_x32(taddr + 32, v1);
  tmem_wait_ld();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t (&u)[32] = x ? v1 : v0;
    if (masked) {
      const uint32_t bits = slot_bits(jb + x * 32, lo, hi);
#pragma unroll
      for (int c = 0; c < 32; ++c) u[c] = (bits & (1u << c)) ? u[c] : 0xff800000u;  // -inf
    }
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const float s0 = __uint_as_float(u[2 * c]), s1 = __uint_as_float(u[2 * c + 1]);
      m[0] = fmaxf(m[0], s0);
      m[1] = fmaxf(m[1], s1);
      const float p0 = fast_exp2(fmaf(s0, scale_log2, neg_m)), p1 = fast_exp2(fmaf(s1, scale_log2, neg_m));
      s[0] += p0;
      s[1] += p1;
      pk[x * 16 + c] = pack_bf16x2(p0, p1);
    }
  }
  sum = s[0] + s[1];
  return fmaxf(m[0], m[1]) * scale_log2;
}
// COLS columns of O times alpha, in tensor memory
template <int COLS>
__device__ __forceinline__ void chunk_rescale(uint32_t taddr, float alpha) {
#pragma unroll 1
  for (int c = 0; c < COLS; c += 32) {
    uint32_t o[32];
    tmem_ld_x32(taddr + c, o);
    tmem_wait_ld();
#pragma unroll
    for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
    tmem_st_x32(taddr + c, o);
  }
}
// rows of a boundary tile of V (slabs of `slabs` x 64 dimensions, 128 keys each) that no row of the item sees
__device__ __forceinline__ void chunk_clear(uint8_t* v, int slabs, int t, const ChunkSeg& g, int lane) {
  for (int x = lane; x < PG_TILE * slabs * 8; x += 32) {
    const int key = (x >> 3) % PG_TILE, slab = (x >> 3) / PG_TILE, j = t * PG_TILE + key;
    if (j < g.lo || j >= g.hi) *reinterpret_cast<uint4*>(v + slab * PG_TILE * 128 + sw128_offset(key, x & 7)) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
}
__device__ __forceinline__ bool chunk_edge(const ChunkSeg& g, int t) { return t * PG_TILE < g.lo || (t + 1) * PG_TILE > g.hi; }

// unit counts of the sequences, and for the join their sum
__device__ __forceinline__ int chunk_units(const PagedSeqs& s, const PagedAttnArgs& a, int* pre, int* status) {
  paged_item_prefix(s.B, pre, CHUNK_THREADS, [&](int b) {
    PagedSeq q;
    return chunk_seq(s, a, b, q, status) ? chunk_cut(q, a).units : 0;
  });
  int total = pre[s.B];
  if (total > a.max_units) {  // rows of q that several sequences claim: more units than n rows can make
    total = a.max_units;
    atomicCAS(status, 0, ST_BAD_INDEX);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_units = total;
  return total;
}

// ---------------------------------------------------------------- D 256: CTA pairs
//   warp 0      TMA loads of this CTA's 64 keys of K
//   warp 1      owns tensor memory; the leader's lane issues S = Q K^T (M = 256) into one of two buffers and O += P V; S of tile t + 1
//               before P V of tile t. A queued product blocks its issue slot until the pipe takes it, so whatever can be waited for
//               earlier is (V before S), and a product's one commit serves the softmax and the copies: S done = its K stage free
//   warps 4-11  softmax: thread = row, group A the first 64 keys of the tile, group B the others; maxima exchanged in shared memory
//   warp 2      TMA loads of Q and of this CTA's half of V's dimensions (all 128 keys)
//   warp 3      in a tile with slots that no row of the item sees (a page's end, the front of a window) it waits for the copy of V
//               and clears those rows, while warp 2 goes on: P is 0 there, but 0 * inf is not. It also plans the segments
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
paged_pair_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const PagedSeqs s, const PagedAttnArgs a, int* __restrict__ status) {
  constexpr int D = 256;
  using L = ChunkSmem<D>;
  constexpr int SLABS = L::SLABS, NS = L::NS, V_SLABS = SLABS / 2;
  constexpr uint32_t IDESC_S = make_idesc(FMT_BF16, FMT_BF16, 256, 128, 0, 0);
  constexpr uint32_t IDESC_O = make_idesc(FMT_BF16, FMT_BF16, 256, D, 0, 1);  // B = V, MN-major (head dimensions contiguous)

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;        // NS
  uint64_t* v_full = k_full + NS;     // NS
  uint64_t* s_done = v_full + NS;     // NS: S of a tile is there, its K stage is free
  uint64_t* o_done = s_done + NS;     // NS: P V of a tile is done, its V stage is free
  uint64_t* v_edge = o_done + NS;     // NS: a boundary tile's copies complete on the CTA's own barrier
  uint64_t* p_ready = v_edge + NS;
  uint64_t* o_free = p_ready + 1;
  uint64_t* seg_full = o_free + 1;    // SEGS
  uint64_t* seg_empty = seg_full + L::SEGS;
  uint32_t* tmem_base_p = reinterpret_cast<uint32_t*>(seg_empty + L::SEGS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_p + 1);
  float* xchg = reinterpret_cast<float*>(smem + L::XCHG_OFF);
  int* pre = reinterpret_cast<int*>(smem + L::PRE_OFF);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx wc{abort_flag, status};
  const uint32_t rank = cluster_ctarank();
  const int n_pairs = static_cast<int>(gridDim.x) >> 1, pair = static_cast<int>(blockIdx.x) >> 1;
  pdl_trigger();
  if (chunk_idle(s, a)) return;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 2);  // one arrival of each CTA: the copies are queued, or the boundary tile is ready
      mbar_init(&s_done[i], 1);
      mbar_init(&o_done[i], 1);
      mbar_init(&v_edge[i], 1);
    }
    mbar_init(p_ready, 16);  // one arrival per softmax warp of both CTAs
    mbar_init(o_free, 16);
    for (int i = 0; i < L::SEGS; ++i) {
      mbar_init(&seg_full[i], 1);
      mbar_init(&seg_empty[i], rank == 0 ? 12 : 11);  // K, V, boundary, 8 softmax warps, and the leader's products
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_base_p, L::TMEM_COLS);
    tmem_relinquish_pair();
  }
  const int total = chunk_units(s, a, pre, status);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before any remote arrival or peer-signalled copy
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_p;
  const int in_page = (1 << s.page_log2) - 1;
  SegRing<L> ring{reinterpret_cast<ChunkSeg*>(smem + L::SEG_OFF), seg_full, seg_empty, 0};
  ChunkSeg g;

  if (warp == 0) {
    const int rl = s.page_log2 < 6 ? s.page_log2 : 6, rows = 1 << rl;  // rows of a K box
    uint32_t cnt = 0;
    bool ok = true;
    while (ok && ring.next(wc, g)) {
      __syncwarp();
      if (lane == 0) ring.done(); else ++ring.n;
      const int32_t* pages = s.table + g.b * s.table_pitch;
      PageRun run;
      run.start(s, pages, g, static_cast<int>(rank) * CH_KH, 6 - rl, rl, lane, status);
      for (int t = g.ta; t < g.tb && ok; ++t, ++cnt) {
        const uint32_t st = cnt % NS;
        if (lane == 0) {
          ok = mbar_wait(wc, &s_done[st], ((cnt / NS) & 1u) ^ 1u, ST_TIMEOUT_EMPTY);
          if (ok && rank == 0) mbar_expect_tx(&k_full[st], 2 * L::KV);
        }
        const int j0 = t * PG_TILE + static_cast<int>(rank) * CH_KH;
        for (int x = 0; x < CH_KH >> rl; ++x) {
          const int pg = run.get(s, pages, g, lane, status);
          if (lane == 0 && ok) {
            const uint32_t bar = map_to_cta(&k_full[st], 0);
            const int at = (j0 + x * rows) & in_page;
            uint8_t* dst = smem + L::K_OFF + st * L::KV + x * rows * 128;
            if (rows == CH_KH)
              tma_load_5d_pair(dst, &tmK, 0, at, 0, g.g, pg, bar);
            else
              for (int y = 0; y < SLABS; ++y) tma_load_5d_pair(dst + y * CH_KH * 128, &tmK, 0, at, y, g.g, pg, bar);
          }
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      }
    }
    if (*abort_flag && lane == 0)  // bounded wait for copies that may still be in flight (the leader's barriers count both CTAs')
      for (uint32_t c = cnt > static_cast<uint32_t>(NS) ? cnt - NS : 0; c <= cnt; ++c)
        for (int spin = 0; spin < 4096 && !mbar_try_wait(&k_full[c % NS], (c / NS) & 1u); ++spin) {}
  } else if (warp == 2) {
    const int rl = s.page_log2 < 7 ? s.page_log2 : 7, rows = 1 << rl;  // rows of a V box
    uint32_t cnt = 0, seg_n = 0;
    bool ok = true;
    while (ok && ring.next(wc, g)) {
      __syncwarp();
      if (lane == 0) ring.done(); else ++ring.n;
      const int32_t* pages = s.table + g.b * s.table_pitch;
      PageRun run;
      run.start(s, pages, g, 0, 7 - rl, rl, lane, status);
      // Q comes with this warp, not with K's: the next segment's K is then not held back until the last product has read Q
      if (lane == 0) {
        ok = mbar_wait(wc, q_empty, (seg_n & 1u) ^ 1u, ST_TIMEOUT_EMPTY);
        if (ok) {
          if (rank == 0) mbar_expect_tx(q_full, 2 * L::Q_BYTES);
          const int qrows = 128 >> a.hp_log2, row = g.row0 + g.tok0 + static_cast<int>(rank) * qrows;
          for (int hh = 0; hh < 1 << a.hp_log2; ++hh)
            for (int x = 0; x < SLABS; ++x)
              tma_load_2d_pair(smem + x * 128 * 128 + hh * qrows * 128, &tmQ, (g.h0 + hh) * D + x * 64, row, map_to_cta(q_full, 0));
        }
      }
      ++seg_n;
      ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      for (int t = g.ta; t < g.tb && ok; ++t, ++cnt) {
        const uint32_t st = cnt % NS;
        const bool edge = chunk_edge(g, t);
        if (lane == 0) {
          ok = mbar_wait(wc, &o_done[st], ((cnt / NS) & 1u) ^ 1u, ST_TIMEOUT_EMPTY);
          if (ok) {
            if (edge)
              mbar_expect_tx(&v_edge[st], L::KV);
            else if (rank == 0)
              mbar_expect_tx(&v_full[st], 2 * L::KV);
            else
              mbar_arrive_cluster(map_to_cta(&v_full[st], 0));
          }
        }
        for (int x = 0; x < PG_TILE >> rl; ++x) {
          const int pg = run.get(s, pages, g, lane, status);
          if (lane == 0 && ok) {
            const uint32_t bar = map_to_cta(&v_full[st], 0);
            const int at = (t * PG_TILE + x * rows) & in_page;
            uint8_t* dst = smem + L::V_OFF + st * L::KV + x * rows * 128;
            for (int y = 0; y < (rows == PG_TILE ? 1 : V_SLABS); ++y) {
              const int slab = static_cast<int>(rank) * V_SLABS + y;
              if (edge)
                tma_load_5d(dst + y * PG_TILE * 128, &tmV, 0, at, slab, g.g, pg, &v_edge[st]);
              else
                tma_load_5d_pair(dst + y * PG_TILE * 128, &tmV, 0, at, slab, g.g, pg, bar);
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      }
    }
    if (*abort_flag && lane == 0) {
      for (uint32_t c = cnt > static_cast<uint32_t>(NS) ? cnt - NS : 0; c <= cnt; ++c)
        for (int spin = 0; spin < 4096 && !mbar_try_wait(&v_full[c % NS], (c / NS) & 1u); ++spin) {}
      for (int spin = 0; seg_n && spin < 4096 && !mbar_try_wait(q_full, (seg_n - 1) & 1u); ++spin) {}
    }
  } else if (warp == 3) {
    uint32_t cnt = 0, edges[NS];  // boundary tiles each stage has held
#pragma unroll
    for (int i = 0; i < NS; ++i) edges[i] = 0;
    SegPlan<L> planner{smem + L::PLAN_OFF, pair, L::PLAN, total, n_pairs, 0, false};
    bool ok = true;
    for (int i = 0; i + 1 < L::SEGS && ok; ++i) ok = planner.publish(s, a, pre, ring, wc, status);
    while (ok && __all_sync(0xffffffffu, ring.next(wc, g))) {
      __syncwarp();
      if (lane == 0) ring.done(); else ++ring.n;
      for (int t = g.ta; t < g.tb; ++t, ++cnt) {
        if (!chunk_edge(g, t)) continue;
        const uint32_t st = cnt % NS;
        uint32_t turn = 0;
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (static_cast<uint32_t>(i) == st) turn = edges[i]++;
        ok = __all_sync(0xffffffffu, mbar_wait(wc, &v_edge[st], turn & 1u, ST_TIMEOUT_FULL));
        if (!ok) break;
        chunk_clear(smem + L::V_OFF + st * L::KV, V_SLABS, t, g, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_release(map_to_cta(&v_full[st], 0));
      }
      ok = ok && planner.publish(s, a, pre, ring, wc, status);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t q_addr = smem_u32(smem);
      uint32_t kc = 0, gt = 0, seg_n = 0;
      bool ok = true;
      auto issue_s = [&]() {  // S of the next tile into buffer kc & 1; its K is there
        tc_fence_after();
        const uint32_t k_addr = smem_u32(smem + L::K_OFF + (kc % NS) * L::KV);
        const uint32_t d_tmem = tmem_base + (kc & 1u) * 128;
#pragma unroll
        for (int x = 0; x < SLABS; ++x) {
          const uint64_t ad = make_smem_desc_sw128(q_addr + x * 128 * 128, 16, 1024);
          const uint64_t bd = make_smem_desc_sw128(k_addr + x * CH_KH * 128, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f16_ss_pair(d_tmem, ad + 2 * k, bd + 2 * k, IDESC_S, (x | k) != 0);
        }
        umma_commit_pair_both(&s_done[kc % NS]);
        ++kc;
      };
      while (ok && ring.next(wc, g)) {
        ring.done();
        const int n_tiles = g.tb - g.ta;
        ok = mbar_wait(wc, q_full, seg_n & 1u, ST_TIMEOUT_FULL) && mbar_wait(wc, &k_full[kc % NS], (kc / NS) & 1u, ST_TIMEOUT_FULL);
        if (!ok) break;
        issue_s();
        for (int i = 0; i < n_tiles; ++i) {
          const uint32_t gi = gt + i, st = gi % NS;
          ok = i + 1 >= n_tiles || mbar_wait(wc, &k_full[kc % NS], (kc / NS) & 1u, ST_TIMEOUT_FULL);
          ok = ok && mbar_wait(wc, &v_full[st], (gi / NS) & 1u, ST_TIMEOUT_FULL);
          if (!ok) break;
          if (i + 1 < n_tiles)
            issue_s();  // buffer (gi + 1) & 1 last held P of tile gi - 1, whose P V was issued before
          else
            umma_commit_pair_both(q_empty);
          ok = mbar_wait(wc, p_ready, gi & 1u, ST_TIMEOUT_OTHER);
          if (ok && i == 0 && seg_n > 0) ok = mbar_wait(wc, o_free, (seg_n - 1) & 1u, ST_TIMEOUT_OTHER);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = make_smem_desc_sw128(smem_u32(smem + L::V_OFF + st * L::KV), PG_TILE * 128, 1024);
#pragma unroll
          for (int k = 0; k < 8; ++k)  // packed bf16 P: 16 keys per 8 columns, the second group's from column 64 on
            umma_f16_ts_pair(tmem_base + L::O_COL, tmem_base + (gi & 1u) * 128 + (k >> 2) * CH_KH + 8 * (k & 3), vd + 128 * k, IDESC_O, (i | k) != 0);
          umma_commit_pair_both(&o_done[st]);
        }
        gt += n_tiles;
        ++seg_n;
      }
    }
  } else {
    const int wg = (warp - 4) >> 2;
    const int qd = warp & 3;  // TMEM lane quarter of this warp
    const int row = qd * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(qd * 32) << 16;
    uint8_t* stage = smem + L::OUT_OFF + (warp - 4) * 2048;
    const uint32_t p_bar = map_to_cta(p_ready, 0), free_bar = map_to_cta(o_free, 0);
    uint32_t gt = 0;
    while (bar_red_and(1 + qd, 64, ring.next(wc, g))) {  // (two warps share these rows and their barrier: they leave together)
      if (lane == 0) ring.done(); else ++ring.n;
      const int n_tiles = g.tb - g.ta, qrows = 128 >> a.hp_log2;
      const int head = g.h0 + (row >> (7 - a.hp_log2));
      const int tok_first = g.tok0 + static_cast<int>(rank) * qrows, tok = tok_first + (row & (qrows - 1));
      const int hi = g.base + tok, lo = a.window > 0 ? hi - a.window + 1 : 0;  // slots the row sees
      const int hi_min = g.base + tok_first, lo_max = a.window > 0 ? hi_min + qrows - a.window : 0;
      float m_ref = -INFINITY, l_run = 0.f;
      bool alive = true;
      for (int i = 0; i < n_tiles; ++i) {
        const uint32_t gi = gt + i;
        const int jb = (g.ta + i) * PG_TILE + wg * CH_KH;
        bool got = mbar_wait(wc, &s_done[gi % NS], (gi / NS) & 1u, ST_TIMEOUT_TMEM);
        float sc[CH_KH];
        float mx = -INFINITY;
        const uint32_t s_tmem = tmem_base + lane_off + (gi & 1u) * 128 + wg * CH_KH;
        got = __all_sync(0xffffffffu, got);
        if (got) {
          tc_fence_after();
          chunk_scores(sc, s_tmem, jb + CH_KH - 1 > hi_min || jb < lo_max, jb, lo, hi);
          mx = chunk_max(sc);
        }
        float* xq = xchg + (gi & 1u) * 256;
        xq[wg * 128 + row] = mx;
        if (!bar_red_and(1 + qd, 64, got)) { alive = false; break; }  // the two warps that share these rows leave together
        mx = fmaxf(mx, xq[(wg ^ 1) * 128 + row]) * a.scale_log2;
        float alpha = 1.f;
        if (mx - m_ref > CH_RESCALE) {  // false for NaN (-inf minus -inf): a row that has seen nothing yet
          alpha = fast_exp2(m_ref - mx);
          m_ref = mx;
        }
        uint32_t pk[CH_KH / 2];
        l_run = l_run * alpha + chunk_probs(sc, a.scale_log2, m_ref == -INFINITY ? 0.f : -m_ref, pk);
        if (i > 0) {
          const bool done = mbar_wait(wc, &o_done[(gi - 1) % NS], ((gi - 1) / NS) & 1u, ST_TIMEOUT_TMEM);
          if (__any_sync(0xffffffffu, alpha != 1.f) && __all_sync(0xffffffffu, done)) {
            // every P V so far has completed and none is issued until all warps have arrived on p_ready
            tc_fence_after();
            chunk_rescale<D / 2>(tmem_base + lane_off + L::O_COL + wg * (D / 2), alpha);
          }
        }
        __syncwarp();
        tmem_st_x32(s_tmem, pk);  // P over the first 32 columns of the S half this thread has read
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(p_bar);
      }
      if (!alive) break;
      gt += n_tiles;

      // end of the segment: O of this group's half of the columns
      float* xq = xchg + 2 * 256;
      xq[wg * 128 + row] = l_run;
      const bool got = mbar_wait(wc, &o_done[(gt - 1) % NS], ((gt - 1) / NS) & 1u, ST_TIMEOUT_TMEM);
      if (!bar_red_and(1 + qd, 64, got)) break;
      tc_fence_after();
      const float l = l_run + xq[(wg ^ 1) * 128 + row];
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a row that sees nothing: 0; a NaN sum stays NaN
      chunk_store<D, D / 2>(a, g, tmem_base + lane_off + L::O_COL + wg * (D / 2), wg * (D / 2), static_cast<int>(rank), qd, lane, inv, stage, [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(free_bar);
      });
      if (wg == 0) chunk_store_stats(a, g, static_cast<int>(rank), row, tok, head, m_ref, l);
    }
  }

  if (threadIdx.x == 0) pdl_wait();  // the kernels behind this one need what the kernel ahead of it wrote, too
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while its peer may still signal its barriers or read its shared memory
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, L::TMEM_COLS);
  }
}

// ---------------------------------------------------------------- D 128: two tiles of rows in one CTA
// The warps' parts as above; the products go round as P V of tile 0, S of tile 0 for the next keys, P V of tile 1, S of tile 1, so that
// while one tile's softmax works the pipe has the other's products.
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
paged_two_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const PagedSeqs s, const PagedAttnArgs a, int* __restrict__ status) {
  constexpr int D = 128;
  using L = ChunkSmem<D>;
  constexpr int SLABS = L::SLABS, NS = L::NS;
  constexpr uint32_t IDESC_S = make_idesc(FMT_BF16, FMT_BF16, 128, 128, 0, 0);
  constexpr uint32_t IDESC_O = make_idesc(FMT_BF16, FMT_BF16, 128, D, 0, 1);  // B = V, MN-major

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;         // NS
  uint64_t* v_full = k_full + NS;      // NS
  uint64_t* v_edge = v_full + NS;      // NS
  uint64_t* s_done = v_edge + NS;      // [tile][NS]: S is there; tile 1's: the K stage is free as well
  uint64_t* o_done = s_done + 2 * NS;  // [tile][NS]: P V is done; tile 1's: the V stage is free as well
  uint64_t* p_ready = o_done + 2 * NS;  // [tile]
  uint64_t* o_free = p_ready + 2;       // [tile]
  uint64_t* seg_full = o_free + 2;
  uint64_t* seg_empty = seg_full + L::SEGS;
  uint32_t* tmem_base_p = reinterpret_cast<uint32_t*>(seg_empty + L::SEGS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_p + 1);
  int* pre = reinterpret_cast<int*>(smem + L::PRE_OFF);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx wc{abort_flag, status};
  pdl_trigger();
  if (chunk_idle(s, a)) return;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_edge[i], 1);
      for (int x = 0; x < 2; ++x) mbar_init(&s_done[x * NS + i], 1), mbar_init(&o_done[x * NS + i], 1);
    }
    for (int x = 0; x < 2; ++x) mbar_init(&p_ready[x], 4), mbar_init(&o_free[x], 4);
    for (int i = 0; i < L::SEGS; ++i) mbar_init(&seg_full[i], 1), mbar_init(&seg_empty[i], 12);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_base_p, L::TMEM_COLS);
    tmem_relinquish();
  }
  const int total = chunk_units(s, a, pre, status);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_p;
  const int in_page = (1 << s.page_log2) - 1;
  SegRing<L> ring{reinterpret_cast<ChunkSeg*>(smem + L::SEG_OFF), seg_full, seg_empty, 0};
  ChunkSeg g;

  if (warp == 0 || warp == 2) {
    const bool is_k = warp == 0;
    const int rl = s.page_log2 < 7 ? s.page_log2 : 7, rows = 1 << rl;  // rows of a box
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* empty = (is_k ? s_done : o_done) + NS;
    const CUtensorMap* tm = is_k ? &tmK : &tmV;
    uint8_t* stages = smem + (is_k ? L::K_OFF : L::V_OFF);
    uint32_t cnt = 0, seg_n = 0;
    bool ok = true;
    while (ok && ring.next(wc, g)) {
      __syncwarp();
      if (lane == 0) ring.done(); else ++ring.n;
      const int32_t* pages = s.table + g.b * s.table_pitch;
      PageRun run;
      run.start(s, pages, g, 0, 7 - rl, rl, lane, status);
      if (!is_k && lane == 0) {  // (K of the next segment is not held back until the last product has read Q)
        ok = mbar_wait(wc, q_empty, (seg_n & 1u) ^ 1u, ST_TIMEOUT_EMPTY);
        if (ok) {
          mbar_expect_tx(q_full, L::Q_BYTES);
          const int qrows = 128 >> a.hp_log2;
          for (int tile = 0; tile < 2; ++tile)
            for (int hh = 0; hh < 1 << a.hp_log2; ++hh)
              for (int x = 0; x < SLABS; ++x)
                tma_load_2d(smem + tile * (L::Q_BYTES / 2) + x * 128 * 128 + hh * qrows * 128, &tmQ, (g.h0 + hh) * D + x * 64, g.row0 + g.tok0 + tile * qrows, q_full);
        }
      }
      ++seg_n;
      ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      for (int t = g.ta; t < g.tb && ok; ++t, ++cnt) {
        const uint32_t st = cnt % NS;
        const bool edge = !is_k && chunk_edge(g, t);
        uint64_t* bar = edge ? &v_edge[st] : &full[st];
        if (lane == 0) {
          ok = mbar_wait(wc, &empty[st], ((cnt / NS) & 1u) ^ 1u, ST_TIMEOUT_EMPTY);
          if (ok) mbar_expect_tx(bar, L::KV);
        }
        for (int x = 0; x < PG_TILE >> rl; ++x) {
          const int pg = run.get(s, pages, g, lane, status);
          if (lane == 0 && ok) {
            uint8_t* dst = stages + st * L::KV + x * rows * 128;
            for (int y = 0; y < (rows == PG_TILE ? 1 : SLABS); ++y)
              tma_load_5d(dst + y * PG_TILE * 128, tm, 0, (t * PG_TILE + x * rows) & in_page, y, g.g, pg, bar);
          }
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      }
    }
    if (*abort_flag && lane == 0) {  // bounded wait for copies that may still be in flight
      for (uint32_t c = cnt > static_cast<uint32_t>(NS) ? cnt - NS : 0; c <= cnt; ++c)
        for (int spin = 0; spin < 4096 && !mbar_try_wait(&full[c % NS], (c / NS) & 1u); ++spin) {}
      for (int spin = 0; !is_k && seg_n && spin < 4096 && !mbar_try_wait(q_full, (seg_n - 1) & 1u); ++spin) {}
    }
  } else if (warp == 3) {
    uint32_t cnt = 0, edges[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) edges[i] = 0;
    SegPlan<L> planner{smem + L::PLAN_OFF, static_cast<int>(blockIdx.x), L::PLAN, total, static_cast<int>(gridDim.x), 0, false};
    bool ok = true;
    for (int i = 0; i + 1 < L::SEGS && ok; ++i) ok = planner.publish(s, a, pre, ring, wc, status);
    while (ok && __all_sync(0xffffffffu, ring.next(wc, g))) {
      __syncwarp();
      if (lane == 0) ring.done(); else ++ring.n;
      for (int t = g.ta; t < g.tb; ++t, ++cnt) {
        if (!chunk_edge(g, t)) continue;
        const uint32_t st = cnt % NS;
        uint32_t turn = 0;
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (static_cast<uint32_t>(i) == st) turn = edges[i]++;
        ok = __all_sync(0xffffffffu, mbar_wait(wc, &v_edge[st], turn & 1u, ST_TIMEOUT_FULL));
        if (!ok) break;
        chunk_clear(smem + L::V_OFF + st * L::KV, SLABS, t, g, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
      }
      ok = ok && planner.publish(s, a, pre, ring, wc, status);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t gt = 0, seg_n = 0;
      bool ok = true;
      auto issue_s = [&](int tile, uint32_t gi) {
        const uint32_t q_addr = smem_u32(smem) + tile * (L::Q_BYTES / 2), k_addr = smem_u32(smem + L::K_OFF + (gi % NS) * L::KV);
#pragma unroll
        for (int x = 0; x < SLABS; ++x) {
          const uint64_t ad = make_smem_desc_sw128(q_addr + x * 128 * 128, 16, 1024);
          const uint64_t bd = make_smem_desc_sw128(k_addr + x * PG_TILE * 128, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f16_ss(tmem_base + tile * 128, ad + 2 * k, bd + 2 * k, IDESC_S, (x | k) != 0);
        }
        umma_commit(&s_done[tile * NS + gi % NS]);
      };
      while (ok && ring.next(wc, g)) {
        ring.done();
        const int n_tiles = g.tb - g.ta;
        ok = mbar_wait(wc, q_full, seg_n & 1u, ST_TIMEOUT_FULL) && mbar_wait(wc, &k_full[gt % NS], (gt / NS) & 1u, ST_TIMEOUT_FULL);
        if (!ok) break;
        tc_fence_after();
        const bool both = g.tok0 + (128 >> a.hp_log2) < g.nq;  // few rows: the second tile has none, and no products
        // S of tile x may replace P of the last segment's end: its P V was issued before
        issue_s(0, gt);
        if (both) issue_s(1, gt);
        else umma_commit(&s_done[NS + gt % NS]);
        for (int i = 0; i < n_tiles && ok; ++i) {
          const uint32_t gi = gt + i, st = gi % NS;
          const bool more = i + 1 < n_tiles;
          ok = mbar_wait(wc, &v_full[st], (gi / NS) & 1u, ST_TIMEOUT_FULL) &&
               (!more || mbar_wait(wc, &k_full[(gi + 1) % NS], ((gi + 1) / NS) & 1u, ST_TIMEOUT_FULL));
          if (!ok) break;
          if (!more) umma_commit(q_empty);
          const uint64_t vd = make_smem_desc_sw128(smem_u32(smem + L::V_OFF + st * L::KV), PG_TILE * 128, 1024);
#pragma unroll
          for (int tile = 0; tile < 2; ++tile) {
            ok = ok && mbar_wait(wc, &p_ready[tile], gi & 1u, ST_TIMEOUT_OTHER);
            if (ok && i == 0 && seg_n > 0) ok = mbar_wait(wc, &o_free[tile], (seg_n - 1) & 1u, ST_TIMEOUT_OTHER);
            if (!ok) break;
            tc_fence_after();
            if (tile == 1 && !both) {  // the copies wait for the second tile's barriers
              umma_commit(&o_done[NS + st]);
              if (more) umma_commit(&s_done[NS + (gi + 1) % NS]);
              break;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)  // packed bf16 P: 16 keys per 8 columns
              umma_f16_ts(tmem_base + L::O_COL + tile * D, tmem_base + tile * 128 + (k >> 2) * CH_KH + 8 * (k & 3), vd + 128 * k, IDESC_O, (i | k) != 0);
            umma_commit(&o_done[tile * NS + st]);
            if (more) issue_s(tile, gi + 1);
          }
        }
        gt += n_tiles;
        ++seg_n;
      }
    }
  } else {
    const int tile = (warp - 4) >> 2;
    const int qd = warp & 3;
    const int row = qd * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(qd * 32) << 16;
    uint8_t* stage = smem + L::OUT_OFF + (warp - 4) * 2048;
    const uint32_t s_tmem = tmem_base + lane_off + tile * 128, o_tmem = tmem_base + lane_off + L::O_COL + tile * D;
    uint32_t gt = 0;
    bool alive = true;
    while (alive && __all_sync(0xffffffffu, ring.next(wc, g))) {
      __syncwarp();
      if (lane == 0) ring.done(); else ++ring.n;
      const int n_tiles = g.tb - g.ta, qrows = 128 >> a.hp_log2;
      const int head = g.h0 + (row >> (7 - a.hp_log2));
      const int tok_first = g.tok0 + tile * qrows, tok = tok_first + (row & (qrows - 1));
      const int hi = g.base + tok, lo = a.window > 0 ? hi - a.window + 1 : 0;
      const int hi_min = g.base + tok_first, lo_max = a.window > 0 ? hi_min + qrows - a.window : 0;
      float m_ref = -INFINITY, l_run = 0.f;
      for (int i = 0; i < n_tiles; ++i) {
        const uint32_t gi = gt + i;
        const int jb = (g.ta + i) * PG_TILE;
        alive = __all_sync(0xffffffffu, mbar_wait(wc, &s_done[tile * NS + gi % NS], (gi / NS) & 1u, ST_TIMEOUT_TMEM));
        if (!alive) break;
        tc_fence_after();
        if (tok_first >= g.nq) {  // no rows in this tile: only the barriers' phases are kept
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[tile]);
          continue;
        }
        const bool masked = jb + PG_TILE - 1 > hi_min || jb < lo_max;
        // p against the reference maximum as it stands, the scores' own maximum found on the way: no pass over the scores before the
        // exponentials. Only where a row outgrew the threshold (or has no maximum yet) is the half done again. The reference is a whole
        // number, so what was computed against the old one is scaled by a power of two, exactly.
        float alpha = 1.f;
#pragma unroll 1
        for (int half = 1; half >= 0; --half) {
          uint32_t pk[32];
          float sum;
          const uint32_t at = s_tmem + half * CH_KH;
          const int jh = jb + half * CH_KH;
          const float mx = chunk_half(at, masked, jh, lo, hi, a.scale_log2, m_ref == -INFINITY ? 0.f : -m_ref, pk, sum);
          const bool grown = mx - m_ref > CH_RESCALE;  // false for NaN (-inf minus -inf): a row that has seen nothing yet
          if (__any_sync(0xffffffffu, grown)) {
            float f = 1.f;
            if (grown) {
              const float m_new = ceilf(mx);
              f = fast_exp2(m_ref - m_new);
              m_ref = m_new;
            }
            alpha *= f;
            l_run *= f;
            if (half == 0) {  // the other half's P is in tensor memory already
              const uint32_t f2 = pack_bf16x2(f, f);
              tmem_wait_st();
              tmem_ld_x32(at + CH_KH, pk);
              tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < 32; ++c) pk[c] = bf2_mul(pk[c], f2);
              tmem_st_x32(at + CH_KH, pk);
            }
            chunk_half(at, masked, jh, lo, hi, a.scale_log2, m_ref == -INFINITY ? 0.f : -m_ref, pk, sum);
          }
          l_run += sum;
          __syncwarp();
          tmem_st_x32(at, pk);  // over the scores this thread has read
        }
        // (S of this tile was issued behind P V of the last: that has completed, and none is in flight until this warp has arrived)
        if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) chunk_rescale<D>(o_tmem, alpha);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[tile]);
      }
      if (!alive) break;
      gt += n_tiles;
      alive = __all_sync(0xffffffffu, mbar_wait(wc, &o_done[tile * NS + (gt - 1) % NS], ((gt - 1) / NS) & 1u, ST_TIMEOUT_TMEM));
      if (!alive) break;
      tc_fence_after();
      if (tok_first >= g.nq) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[tile]);
        continue;
      }
      const float inv = l_run > 0.f ? 1.f / l_run : (l_run == 0.f ? 0.f : l_run);
      chunk_store<D, D>(a, g, o_tmem, 0, tile, qd, lane, inv, stage, [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[tile]);
      });
      chunk_store_stats(a, g, tile, row, tok, head, m_ref, l_run);
    }
  }

  if (threadIdx.x == 0) pdl_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, L::TMEM_COLS);
  }
}

// ---------------------------------------------------------------- join of the cut items
// CTAs (x, y) over units `it`: the item that the unit is the first to begin inside of, as the planning warps have left word; 16 of its 256 rows, a
// warp per row, the pieces added in the order of the units (an item in nine parts is a chain of loads for a row, so rows side by side)
static constexpr int JOIN_ROWS = 16;
template <int D, int SLOTS>  // of 256 rows a unit has
__global__ void __launch_bounds__(256) paged_chunk_join_kernel(const PagedSeqs s, const PagedAttnArgs a, int* __restrict__ status) {
  pdl_trigger();
  pdl_wait();
  constexpr int V = D / 128;  // float4 per lane
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int APART = SLOTS * 256;  // rows between an item's further pieces
  const int total = *a.n_units, ql = 7 - a.hp_log2;
  for (int it = blockIdx.x; it < total; it += gridDim.x) {
    const ChunkJoin join = a.joins[it];
    if (join.pieces == 0) continue;
    const int last = it + join.pieces - 2 < a.max_units ? join.pieces - 2 : a.max_units - 1 - it;
    const int64_t first = static_cast<int64_t>(join.first) * 256;
    for (int r = blockIdx.y * JOIN_ROWS + warp; r < (blockIdx.y + 1) * JOIN_ROWS; r += 8) {
      const int in = r & 127, tok = join.tok0 + ((r >> 7) << ql) + (in & ((1 << ql) - 1)), head = join.h0 + (in >> ql);
      if (tok >= join.nq) continue;
      const int64_t at0 = first + r, at = static_cast<int64_t>(it) * APART + r;
      float m = a.chunk_ml[at0].x;
#pragma unroll 4
      for (int y = 0; y <= last; ++y) m = fmaxf(m, a.chunk_ml[at + y * APART].x);
      int splits = 0;  // the row's own, behind the front it shares
      int64_t own = 0, own_step = 0;
      if (join.b1) {
        int b = join.b0 - 1;  // the last sequence that begins at or before the row (the lanes look at 32 at a time: no chain of loads)
        for (int b0 = join.b0; b0 < join.b1; b0 += 32) b += __popc(__ballot_sync(0xffffffffu, b0 + lane < join.b1 && s.cu[b0 + lane] <= join.row0 + tok));
        const PagedSeq q = paged_seq(s, b, status);
        const int all = q.nq * a.group;
        splits = attn_cut(q, a).splits;
        own_step = static_cast<int64_t>(a.h) * all;
        own = b * a.seq_parts + static_cast<int64_t>(head / a.group) * all + (join.row0 + tok - q.row0) * a.group + head % a.group;
        for (int y = 0; y < splits; ++y) m = fmaxf(m, a.part_ml[own + y * own_step].x);
      }
      const float neg_m = m == -INFINITY ? 0.f : -m;
      float l = 0.f;
      float4 acc[V];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int y = -1; y <= last; ++y) {
        const int64_t from = y < 0 ? at0 : at + y * APART;
        const float2 ml = a.chunk_ml[from];
        const float f = fast_exp2(ml.x + neg_m);
        l = fmaf(f, ml.y, l);
        const float4* src = reinterpret_cast<const float4*>(a.chunk_o + from * D);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float4 z = src[v * 32 + lane];
          acc[v].x = fmaf(f, z.x, acc[v].x), acc[v].y = fmaf(f, z.y, acc[v].y), acc[v].z = fmaf(f, z.z, acc[v].z), acc[v].w = fmaf(f, z.w, acc[v].w);
        }
      }
#pragma unroll 2
      for (int y = 0; y < splits; ++y) {
        const int64_t from = own + y * own_step;
        const float2 ml = a.part_ml[from];
        const float f = fast_exp2(ml.x + neg_m);
        l = fmaf(f, ml.y, l);
        const float4* src = reinterpret_cast<const float4*>(a.part_o + from * D);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float4 z = src[v * 32 + lane];
          acc[v].x = fmaf(f, z.x, acc[v].x), acc[v].y = fmaf(f, z.y, acc[v].y), acc[v].z = fmaf(f, z.z, acc[v].z), acc[v].w = fmaf(f, z.w, acc[v].w);
        }
      }
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      __nv_bfloat16* dst = a.out + (join.row0 + tok) * a.out_pitch + static_cast<int64_t>(head) * D;
#pragma unroll
      for (int v = 0; v < V; ++v)
        *reinterpret_cast<uint2*>(dst + (v * 32 + lane) * 4) =
            make_uint2(pack_bf16x2(acc[v].x * inv, acc[v].y * inv), pack_bf16x2(acc[v].z * inv, acc[v].w * inv));
      if (a.lse && lane == 0) a.lse[static_cast<int64_t>(join.row0 + tok) * a.H + head] = m + log2f(l);
    }
  }
}

// ---------------------------------------------------------------- the keys' attention weights of a chunk
// weights_out[j] = decay weights_in[j] + sum over rows p(row, j), p = exp2(s scale - lse(row)), with the rows' lse from above: a second
// pass over Q K^T, this time with the keys as the rows of the product, so that a key's sum stays in one thread: S^T = K Q^T, thread =
// key, 64 query rows a stage along its columns. No reduction across threads, no atomics: a key adds its rows in one fixed order.
// Item = 256 keys of a (sequence, kv head), both tiles of K resident in shared memory while the rows that see any of them stream by.
// Bound by the exponentials and what surrounds them (256 x 64 a stage at 16 per cycle and SM: 1 024 cycles, the products 512 at D 128
// and 1 024 at D 256; measured 2 050 a stage: reading S out of tensor memory and the instructions around each exponential share the
// issue slots). 1 024 tokens over 8 192 (32 / 16 heads of 128): 295 us with the attention, about 137 of them here; scores kept in memory
// and read back took 2 500 for the same.
template <int D>
struct ChunkWeightSmem {
  static constexpr int SLABS = D / 64;
  static constexpr int K_TILE = SLABS * 128 * 128;  // 128 keys
  static constexpr int NK = D == 256 ? 1 : 2;       // items whose keys are held (or being fetched)
  static constexpr int Q_STAGE = SLABS * 64 * 128;  // 64 rows of q
  static constexpr int NQ = D == 256 ? 2 : 4;
  static constexpr int NS = 4;                      // S buffers of 128 columns, each with its rows' lse
  static constexpr int Q_OFF = NK * 2 * K_TILE;
  static constexpr int LSE_OFF = Q_OFF + NQ * Q_STAGE;
  static constexpr int BAR_OFF = LSE_OFF + NS * 64 * 4;
  static constexpr int PRE_OFF = BAR_OFF + 256;
  static constexpr int TOTAL = PRE_OFF + (PG_MAX_SEQS + 2) * 4 + 1024;
};
static_assert(ChunkWeightSmem<256>::TOTAL <= 232448 && ChunkWeightSmem<128>::TOTAL <= 232448, "shared memory of a CTA");
static constexpr int CHUNK_WEIGHT_THREADS = 352;

struct ChunkWeightItem {
  PagedSeq q;
  int b, g, j0;          // first key
  int hp, tok, sets;     // heads and tokens of a stage of 64 rows, head sets of the kv head
  int tt0, tt1;          // token tiles with rows that see some of the keys
};
__device__ __forceinline__ ChunkWeightItem chunk_weight_item(const PagedSeqs& s, const PagedAttnArgs& a, const int* pre, int it, int* status) {
  ChunkWeightItem w;
  w.b = paged_find(pre, s.B, it);
  w.q = paged_seq(s, w.b, status);
  const int x = it - pre[w.b];
  w.g = x % a.h;
  w.j0 = x / a.h * 256;
  w.hp = 1 << a.hp_log2;
  w.tok = 64 >> a.hp_log2;
  w.sets = a.sets;
  const int base = w.q.len - w.q.nq;
  const int first = w.j0 > base ? w.j0 - base : 0;  // tokens before it sit before every key
  int end = w.q.nq;
  if (a.window > 0) {
    const int64_t e = static_cast<int64_t>(w.j0) + 255 + a.window - base;  // tokens from it on see none of the keys
    end = e < end ? (e > 0 ? static_cast<int>(e) : 0) : end;
  }
  w.tt0 = first / w.tok;
  w.tt1 = end > first ? (end + w.tok - 1) / w.tok : w.tt0;
  return w;
}

// A row's lse as it is subtracted from its scores, hidden ones of which are -inf: their p has to come out as 0 whatever the lse is. A row
// whose scores are all -inf weighs nothing (exp2(-inf - inf) = 0). One whose sum is NaN gets the lowest number instead: the slots it sees become
// infinite, which no sum of p is (weight_sum makes it NaN again), and a hidden score of -inf stays -inf.
static constexpr float NAN_LSE = -3.402823466e38f;
__device__ __forceinline__ float weight_lse(float x) { return x != x ? NAN_LSE : x == -INFINITY ? INFINITY : x; }
__device__ __forceinline__ float weight_sum(float x) { return x == INFINITY ? NAN : x; }

template <int D>
__global__ void __launch_bounds__(CHUNK_WEIGHT_THREADS, 1)
paged_chunk_weight_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const PagedSeqs s, const PagedAttnArgs a,
                          const PagedWeightArgs wa, int* __restrict__ status) {
  using L = ChunkWeightSmem<D>;
  constexpr int SLABS = L::SLABS, NK = L::NK, NQ = L::NQ, NS = L::NS;
  constexpr uint32_t IDESC = make_idesc(FMT_BF16, FMT_BF16, 128, 64, 0, 0);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* k_empty = k_full + NK;
  uint64_t* q_full = k_empty + NK;
  uint64_t* q_empty = q_full + NQ;
  uint64_t* s_full = q_empty + NQ;
  uint64_t* s_empty = s_full + NS;
  uint64_t* lse_full = s_empty + NS;
  uint32_t* tmem_base_p = reinterpret_cast<uint32_t*>(lse_full + NS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_p + 1);
  float* lse_ring = reinterpret_cast<float*>(smem + L::LSE_OFF);
  int* pre = reinterpret_cast<int*>(smem + L::PRE_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx wc{abort_flag, status};
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < NK; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < NQ; ++i) mbar_init(&q_full[i], 1), mbar_init(&q_empty[i], 1);
    for (int i = 0; i < NS; ++i) mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], 8), mbar_init(&lse_full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
  }
  if (warp == 1) {
    tmem_alloc(tmem_base_p, 512);
    tmem_relinquish();
  }
  paged_item_prefix(s.B, pre, CHUNK_WEIGHT_THREADS, [&](int b) {
    const PagedSeq q = paged_seq(s, b, status);
    return a.only == 3 || chunk_class(q, a) ? a.h * ((q.len + 255) / 256) : 0;  // (alone in the call: also without new rows)
  });
  const int total = pre[s.B];
  pdl_wait();  // lse is the kernels' ahead
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_p;
  const int in_page = (1 << s.page_log2) - 1;

  if (warp == 0) {
    if (lane == 0) {
      const int rows = s.page_log2 < 7 ? 1 << s.page_log2 : PG_TILE;
      uint32_t n = 0;
      for (int it = blockIdx.x; it < total; it += gridDim.x) {
        const ChunkWeightItem w = chunk_weight_item(s, a, pre, it, status);
        if (w.tt0 >= w.tt1) continue;  // keys that no row sees: only the decay is left
        const int32_t* pages = s.table + w.b * s.table_pitch;
        const uint32_t st = n % NK;
        if (!mbar_wait(wc, &k_empty[st], ((n / NK) & 1u) ^ 1u, ST_TIMEOUT_EMPTY)) break;
        mbar_expect_tx(&k_full[st], 2 * L::K_TILE);
        for (int t = 0; t < 2; ++t)
          for (int x = 0; x < PG_TILE / rows; ++x) {
            const int j = w.j0 + t * PG_TILE + x * rows;
            const int pg = chunk_page(s, pages, j, rows, 0, w.q.len, status);
            uint8_t* dst = smem + (st * 2 + t) * L::K_TILE + x * rows * 128;
            for (int y = 0; y < (rows == PG_TILE ? 1 : SLABS); ++y) tma_load_5d(dst + y * PG_TILE * 128, &tmK, 0, j & in_page, y, w.g, pg, &k_full[st]);
          }
        ++n;
      }
      if (*abort_flag)  // bounded wait for copies that may still be in flight
        for (uint32_t c = n > static_cast<uint32_t>(NK) ? n - NK : 0; c < n; ++c)
          for (int spin = 0; spin < 4096 && !mbar_try_wait(&k_full[c % NK], (c / NK) & 1u); ++spin) {}
    }
  } else if (warp == 10) {
    uint32_t n = 0;
    bool ok = true;
    for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
      const ChunkWeightItem w = chunk_weight_item(s, a, pre, it, status);
      // lse of the stage's rows r and r + 32, fetched a stage ahead (nothing looks at it before it is stored)
      const int tl = 6 - a.hp_log2;  // log2 of a head's rows in a stage
      float next[2] = {0.f, 0.f};
      auto fetch = [&](int set, int tt) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = lane + 32 * x, tok = (tt << tl) + (r & ((1 << tl) - 1));
          next[x] = tok < w.q.nq ? a.lse[static_cast<int64_t>(w.q.row0 + tok) * a.H + w.g * a.group + (set << a.hp_log2) + (r >> tl)] : INFINITY;
        }
      };
      if (w.tt0 < w.tt1) fetch(0, w.tt0);
      for (int set = 0; set < w.sets && ok; ++set)
        for (int tt = w.tt0; tt < w.tt1; ++tt, ++n) {
          const uint32_t st = n % NQ, sl = n % NS;
          ok = __all_sync(0xffffffffu, mbar_wait(wc, &q_empty[st], ((n / NQ) & 1u) ^ 1u, ST_TIMEOUT_EMPTY));
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(&q_full[st], L::Q_STAGE);
            for (int hh = 0; hh < w.hp; ++hh)
              for (int x = 0; x < SLABS; ++x)
                tma_load_2d(smem + L::Q_OFF + st * L::Q_STAGE + x * 64 * 128 + hh * w.tok * 128, &tmQ, (w.g * a.group + set * w.hp + hh) * D + x * 64,
                            w.q.row0 + tt * w.tok, &q_full[st]);
          }
          const float v0 = next[0], v1 = next[1];
          if (tt + 1 < w.tt1) fetch(set, tt + 1);
          else if (set + 1 < w.sets) fetch(set + 1, w.tt0);
          ok = __all_sync(0xffffffffu, mbar_wait(wc, &s_empty[sl], ((n / NS) & 1u) ^ 1u, ST_TIMEOUT_EMPTY));
          if (!ok) break;
          lse_ring[sl * 64 + lane] = weight_lse(v0);
          lse_ring[sl * 64 + lane + 32] = weight_lse(v1);
          __syncwarp();
          if (lane == 0) mbar_arrive(&lse_full[sl]);
        }
    }
    if (*abort_flag && lane == 0)
      for (uint32_t c = n > static_cast<uint32_t>(NQ) ? n - NQ : 0; c < n; ++c)
        for (int spin = 0; spin < 4096 && !mbar_try_wait(&q_full[c % NQ], (c / NQ) & 1u); ++spin) {}
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t n = 0, k = 0;
      bool ok = true;
      for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
        const ChunkWeightItem w = chunk_weight_item(s, a, pre, it, status);
        if (w.tt0 >= w.tt1) continue;
        if (!mbar_wait(wc, &k_full[k % NK], (k / NK) & 1u, ST_TIMEOUT_FULL)) break;
        const uint32_t k_addr = smem_u32(smem) + (k % NK) * 2 * L::K_TILE;
        const int stages = w.sets * (w.tt1 - w.tt0);
        for (int i = 0; i < stages; ++i, ++n) {
          if (!mbar_wait(wc, &s_empty[n % NS], ((n / NS) & 1u) ^ 1u, ST_TIMEOUT_TMEM)) { ok = false; break; }
          if (!mbar_wait(wc, &q_full[n % NQ], (n / NQ) & 1u, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t q_addr = smem_u32(smem + L::Q_OFF + (n % NQ) * L::Q_STAGE);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < SLABS; ++x) {
              const uint64_t ad = make_smem_desc_sw128(k_addr + t * L::K_TILE + x * 128 * 128, 16, 1024);
              const uint64_t bd = make_smem_desc_sw128(q_addr + x * 64 * 128, 16, 1024);
#pragma unroll
              for (int y = 0; y < 4; ++y) umma_f16_ss(tmem_base + (n % NS) * 128 + t * 64, ad + 2 * y, bd + 2 * y, IDESC, (x | y) != 0);
            }
          umma_commit(&q_empty[n % NQ]);
          umma_commit(&s_full[n % NS]);
        }
        if (ok) umma_commit(&k_empty[k % NK]);
        ++k;
      }
    }
  } else {
    const int kt = (warp - 2) >> 2, qd = warp & 3;
    const uint32_t lane_off = static_cast<uint32_t>(qd * 32) << 16;
    uint32_t n = 0;
    bool ok = true;
    for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
      const ChunkWeightItem w = chunk_weight_item(s, a, pre, it, status);
      const int j = w.j0 + kt * PG_TILE + qd * 32 + lane, base = w.q.len - w.q.nq;
      const int tile_lo = w.j0 + kt * PG_TILE;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      for (int set = 0; set < w.sets && ok; ++set)
        for (int tt = w.tt0; tt < w.tt1; ++tt, ++n) {
          const uint32_t sl = n % NS;
          ok = mbar_wait(wc, &s_full[sl], (n / NS) & 1u, ST_TIMEOUT_TMEM) && mbar_wait(wc, &lse_full[sl], (n / NS) & 1u, ST_TIMEOUT_FULL);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          uint32_t v0[32], v1[32];
          const uint32_t at = tmem_base + lane_off + sl * 128 + kt * 64;
          tmem_ld_x32(at, v0);
          tmem_ld_x32(at + 32, v1);
          tmem_wait_ld();
          const float4* lse = reinterpret_cast<const float4*>(lse_ring + sl * 64);
          const int slot0 = base + tt * w.tok;  // of the stage's first token
          const int left = w.q.nq - tt * w.tok;  // tokens of the stage that are the sequence's: the rows behind them are a neighbour's or none's
          const bool masked = left < w.tok || slot0 < tile_lo + PG_TILE - 1 || (a.window > 0 && slot0 + w.tok - 1 >= tile_lo + a.window);
          if (masked) {  // hidden scores to -inf ahead of the exponentials: no branch inside the unrolled loop
            const int lo = j - slot0, tm = w.tok - 1;  // tokens [lo, hi) of the stage see the key; w.tok is a power of two
            const int end = a.window > 0 ? lo + a.window : w.tok, hi = end < left ? end : left;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const int t0 = c & tm, t1 = (c + 32) & tm;
              v0[c] = t0 >= lo && t0 < hi ? v0[c] : 0xff800000u;
              v1[c] = t1 >= lo && t1 < hi ? v1[c] : 0xff800000u;
            }
          }
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float4 z = lse[c];
            const uint32_t* v = c < 8 ? &v0[c * 4] : &v1[c * 4 - 32];
            sum[0] += fast_exp2(fmaf(__uint_as_float(v[0]), a.scale_log2, -z.x));
            sum[1] += fast_exp2(fmaf(__uint_as_float(v[1]), a.scale_log2, -z.y));
            sum[2] += fast_exp2(fmaf(__uint_as_float(v[2]), a.scale_log2, -z.z));
            sum[3] += fast_exp2(fmaf(__uint_as_float(v[3]), a.scale_log2, -z.w));
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[sl]);
        }
      if (ok && j < w.q.len) {
        const float old = wa.decay != 0.f ? wa.in[w.b * wa.in_seq + w.g * wa.in_head + j] * wa.decay : 0.f;
        wa.out[w.b * wa.out_seq + w.g * wa.out_head + j] = old + weight_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D>
static int launch_chunk(const PagedPool& kp, const PagedPool& vp, const PagedSeqs& s, const PagedAttnArgs& a, const PagedWeightArgs* w, bool early,
                        cudaStream_t st, int dev, int* status) {
  using L = ChunkSmem<D>;
  CUtensorMap tmQ, tmK, tmV;
  const int hp = 1 << a.hp_log2;
  int r;
  const uint32_t krows = kp.page < CH_KH ? static_cast<uint32_t>(kp.page) : static_cast<uint32_t>(CH_KH);
  const uint32_t vrows = kp.page < PG_TILE ? static_cast<uint32_t>(kp.page) : static_cast<uint32_t>(PG_TILE);
  if ((r = make_tmap_2d(&tmQ, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.q, s.n, static_cast<uint64_t>(a.H) * D, a.q_pitch * 2, 64, 128 / hp))) return r;
  if (D == 256) {  // a CTA's 64 keys of K, its half of V's dimensions
    if ((r = make_tmap_pages(&tmK, kp, krows, krows == CH_KH ? D / 64 : 1)) || (r = make_tmap_pages(&tmV, vp, vrows, vrows == PG_TILE ? D / 128 : 1))) return r;
  } else if ((r = make_tmap_pages(&tmK, kp, vrows, vrows == PG_TILE ? D / 64 : 1)) || (r = make_tmap_pages(&tmV, vp, vrows, vrows == PG_TILE ? D / 64 : 1))) {
    return r;
  }
  auto kern = D == 256 ? paged_pair_kernel : paged_two_kernel;
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    SPINF_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL));
    SPINF_CUDA_OK(cudaFuncSetAttribute(paged_chunk_weight_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkWeightSmem<D>::TOTAL));
    attr_set[dev].store(true, std::memory_order_release);
  }
  SPINF_CUDA_OK(launch_after(kern, dim3(static_cast<unsigned>(D == 256 ? sm_count() / 2 * 2 : sm_count())), dim3(CHUNK_THREADS), st, L::TOTAL,
                             D == 256 ? 2 : 1, early, tmQ, tmK, tmV, s, a, status));
  const auto join = a.unit_slots == 1 ? paged_chunk_join_kernel<D, 1> : paged_chunk_join_kernel<D, 2>;
  SPINF_CUDA_OK(launch_after(join, dim3(static_cast<unsigned>(a.max_units < PG_SMS ? a.max_units : PG_SMS), 256 / JOIN_ROWS), dim3(256), st, 0, 1, true, s, a, status));
  if (!w) return 0;
  CUtensorMap tmQw, tmKw;
  if ((r = make_tmap_2d(&tmQw, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.q, s.n, static_cast<uint64_t>(a.H) * D, a.q_pitch * 2, 64, 64 / hp))) return r;
  if ((r = make_tmap_pages(&tmKw, kp, vrows, vrows == PG_TILE ? D / 64 : 1))) return r;
  SPINF_CUDA_OK(launch_after(paged_chunk_weight_kernel<D>, dim3(static_cast<unsigned>(sm_count())), dim3(CHUNK_WEIGHT_THREADS), st, ChunkWeightSmem<D>::TOTAL, 1, true,
                             tmQw, tmKw, s, a, *w, status));
  return 0;
}

int paged_chunk_launch(int D, const PagedPool& kp, const PagedPool& vp, const PagedSeqs& s, const PagedAttnArgs& a, const PagedWeightArgs* w, bool early,
                       cudaStream_t st, int dev, int* status) {
  return D == 256 ? launch_chunk<256>(kp, vp, s, a, w, early, st, dev, status) : launch_chunk<128>(kp, vp, s, a, w, early, st, dev, status);
}

}  // namespace spinf
