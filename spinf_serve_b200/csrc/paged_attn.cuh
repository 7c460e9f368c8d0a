// The paged attention's arguments and the rules by which its kernels share out a call: which kernel takes a sequence, and how the
// sequence's work is cut. All rules look at the sequence's own lengths and the model's heads only.
#pragma once
#include "paged.cuh"

namespace spinf {

struct ChunkJoin;

struct PagedAttnArgs {
  const __nv_bfloat16* q;
  int64_t q_pitch;
  __nv_bfloat16* out;
  int64_t out_pitch;
  int H, h, D, group, window;
  int hp_log2, sets;  // chunk kernels: heads of an item, items of a kv head and token tile
  float scale_log2;
  int only;        // one sequence in the call: the kernel its row limit asks for (1 step, 2 few rows, 3 chunk) takes it; 0: by rows
  int chunk_rows;  // sequences with more query rows per kv head than this are the chunk kernel's
  // split keys, few rows: part_o [B][seq_parts][D], part_ml [B][seq_parts] (maximum in log2 units, sum)
  float* part_o;
  float2* part_ml;
  int64_t seq_parts;
  // cut items of the chunk kernel: 256 rows once or twice per unit, and what to join
  int unit_slots;
  float* chunk_o;
  float2* chunk_ml;
  ChunkJoin* joins;  // [max_units]
  int32_t* n_units;
  int max_units;  // units there is room for
  float* lse;     // [n][H] log2 units, or null: what the weights are normalised with
  float* scores;  // [B][tok_cap][H][score_pitch] log2 units, or null: kept for the weights
  int64_t score_pitch;
  int tok_cap;
  int fronts_only;  // no sequence of the call can be a chunk: the chunk kernels have the groups' fronts only
};

struct PagedWeightArgs {
  const float* in;  // [B][h][cap] fp32
  float* out;
  int64_t in_seq, in_head, out_seq, out_head;  // strides
  float decay;                                 // 0: `in` is not read
};

static constexpr int RT = 64;         // query rows of an item of the few-row kernel
static constexpr int STEP_ROWS = 16;  // rows per kv head a decoding step's kernel takes

__host__ __device__ inline int class_of(int64_t rows, int chunk_rows) { return rows <= STEP_ROWS ? 1 : rows > chunk_rows ? 3 : 2; }
__device__ __forceinline__ int seq_class(const PagedSeq& q, const PagedAttnArgs& a) {
  if (q.nq == 0 || a.only) return q.nq == 0 ? 0 : a.only;
  const int c = class_of(q.nq * a.group, a.chunk_rows);
  return c == 3 && q.skip ? 2 : c;  // (behind a front that a group shares little is left: few-row work)
}
__device__ __forceinline__ bool step_class(const PagedSeq& q, const PagedAttnArgs& a) { return seq_class(q, a) == 1; }
__device__ __forceinline__ bool rows_class(const PagedSeq& q, const PagedAttnArgs& a) { return seq_class(q, a) == 2; }
__device__ __forceinline__ bool chunk_class(const PagedSeq& q, const PagedAttnArgs& a) { return seq_class(q, a) == 3; }
__device__ __forceinline__ PagedCut step_cut(const PagedSeq& q, const PagedAttnArgs& a) { return paged_cut(q, a.window, 1, a.h, PG_SMS, 1); }
// Splits of at least two tiles: shorter ones answer few sequences sooner and cost many more, since every split leaves up to 64 rows of
// partial results (12 new tokens, 24 / 4 heads of 256, splits of at least 4 / 2 / 1 tiles: one sequence of 2 048 38 / 27 / 21 us, 16 of them
// 148 / 168 / 195, 56 of them 441 / 537 / 628).
__device__ __forceinline__ PagedCut rows_cut(const PagedSeq& q, const PagedAttnArgs& a) {
  const int rt = (q.nq * a.group + RT - 1) / RT;
  return paged_cut(q, a.window, rt, a.h * rt, PG_SMS, 2);
}
__device__ __forceinline__ PagedCut attn_cut(const PagedSeq& q, const PagedAttnArgs& a) { return step_class(q, a) ? step_cut(q, a) : rows_cut(q, a); }

// ---- the chunk kernel: items of 256 rows (hp heads x 256 / hp tokens), their key tiles dealt out in equal units
// units of a sequence: one per CTA pair (D 256) or CTA (D 128)
__host__ __device__ constexpr int chunk_units_of(int D) { return D == 256 ? PG_SMS / 2 : PG_SMS; }
static constexpr int CHUNK_MIN_TILES = 8;       // least (item, tile) pairs of a unit that begins anywhere: below that a cut costs more than it spreads
static constexpr int CHUNK_SHORT = 24;          // key tiles of an item that is not worth cutting where there are items enough

// heads of an item, as a power of two: the largest that divides the group, at most 8 (16 rows of a head in one tile); more heads per
// item mean fewer tokens, so less of the causal triangle is padding
__host__ __device__ constexpr int chunk_heads_log2(int group) { return group % 8 == 0 ? 3 : group % 4 == 0 ? 2 : group % 2 == 0 ? 1 : 0; }

struct ChunkCut {
  int tok_log2, ntt, per_tt;  // tokens of an item, token tiles, items of a token tile
  int work;                   // (item, key tile) pairs
  int units, quot, rem;       // unit u takes quot pairs, the first `rem` units one more
  bool whole;                 // units take whole items: those that begin in their range
  int parts;                  // not 0: no more items than the GPU runs at once, every unit is one of the `parts` equal parts of an item

  __device__ __forceinline__ void slots(const PagedSeq& q, const PagedAttnArgs& a, int tt, int& lo, int& hi) const {
    const int base = q.len - q.nq, first = base + (tt << tok_log2);
    const int end = (tt + 1) << tok_log2 < q.nq ? base + ((tt + 1) << tok_log2) : q.len;
    lo = a.window > 0 && first - a.window + 1 > 0 ? first - a.window + 1 : 0;
    hi = end > 0 ? end : 0;
    hi = hi < q.cap ? hi : q.cap;
  }
  // key tiles [t0, t0 + nt) of a token tile; one (fully masked) where nothing is seen, so that its rows are written
  __device__ __forceinline__ void tiles(const PagedSeq& q, const PagedAttnArgs& a, int tt, int& t0, int& nt) const {
    int lo, hi;
    slots(q, a, tt, lo, hi);
    t0 = lo >> 7;
    nt = ((hi + PG_TILE - 1) >> 7) - t0;
    nt = nt > 0 ? nt : 1;
  }
  __device__ __forceinline__ int begin(int u) const { return u * quot + (u < rem ? u : rem); }
  __device__ __forceinline__ int unit_of(int w) const {
    const int edge = rem * (quot + 1);
    return w < edge ? w / (quot + 1) : rem + (w - edge) / quot;
  }
};
static_assert(PG_TILE == 128, "key tiles are counted by shifts");
__device__ __forceinline__ ChunkCut chunk_cut(const PagedSeq& q, const PagedAttnArgs& a) {
  ChunkCut c;
  c.tok_log2 = 8 - a.hp_log2;
  c.ntt = (q.nq + (1 << c.tok_log2) - 1) >> c.tok_log2;
  c.per_tt = a.H >> a.hp_log2;
  int tiles = 0;
#pragma unroll 1
  for (int tt = 0; tt < c.ntt; ++tt) {
    int t0, nt;
    c.tiles(q, a, tt, t0, nt);
    tiles += nt;
  }
  c.work = tiles * c.per_tt;  // (the host has checked that this fits)
  const int most = chunk_units_of(a.D), items = c.ntt * c.per_tt;
  const bool brief = tiles <= CHUNK_SHORT * c.ntt, front = q.cap != PG_NO_CAP;
  c.parts = 0;
  c.whole = false;
  if (front || (items <= most && (c.ntt == 1 || brief))) {
    // few items: one unit each, or (a single token tile; a group's front, whose items are all alike) as many equal parts as there is
    // room for, of at least four tiles
    int k = 1;
    if (c.ntt == 1 || front) {
      const int each = tiles / c.ntt / 4;
      k = most / items;
      k = k < each ? k : each;
      k = k > 1 ? k : 1;
    }
    c.parts = k;
    c.units = items * k;
    c.quot = c.rem = 0;
    return c;
  }
  const int u = c.work / CHUNK_MIN_TILES;
  c.units = u < 1 ? 1 : u > most ? most : u;
  c.quot = c.work / c.units;
  c.rem = c.work - c.quot * c.units;
  c.whole = brief && 2 * items >= most;  // many short items (a window): a cut would cost about as much as the imbalance it removes
  return c;
}

// what the join has to do for a unit that is the first to begin inside of an item (pieces 0: nothing)
struct alignas(16) ChunkJoin {
  int pieces;             // partial results of the item, the first of them not the unit's own
  int first;              // the one before (in units of 256 rows); the others are 2 it, 2 it + 2, ..
  int row0, nq, tok0, h0;
  int b0, b1;             // a group's front: the rows belong to these sequences, whose own splits are joined here, too (b1 = 0: none)
};

// ---- the common front of neighbouring sequences (branches of one content): read once for all of their rows, by the chunk kernels, as
// if it were one sequence whose rows see all of it; the sequences' own kernels begin behind it, and the chunk join adds the two.
static constexpr int SHARE_TILES = 8;  // least key tiles of a front (56 sequences of 40 new tokens over 512: 127 us, read together 182; over 1 024: 252, 194)
static constexpr int SHARE_ROWS = 4;   // a group's sequences have up to so many times the rows that make a chunk
// The further kernels cost about 20 us, which the reading they save has to outweigh: measured without / with (us), new tokens over a
// front of that many: 16 / 8 heads of 256, one new token each: 8 over 2 048 (117 MB saved) 36 / 36, 8 over 1 024 (59 MB) 23 / 30, 16
// over 2 048 (252 MB) 60 / 42; twelve new tokens: 6 over 2 048 (84 MB) 47 / 46; 24 / 4 heads of 256, one each: 8 over 4 096 (117 MB)
// 45 / 44; 8 / 8 heads of 128: 8 over 4 096 (117 MB) 31 / 32, 16 over 4 096 (252 MB) 51 / 42. Further up: 56 of 40 new tokens over 4 096
// 796 / 285, 56 of one over 16 384 681 / 118.
__host__ __device__ inline bool share_pays(int64_t seqs, int64_t tokens, int h, int D) { return (seqs - 1) * tokens * h * D * 4 >= 1 << 27; }
// nothing for the chunk kernels: no chunk, and no group found. Their CTAs leave before they set anything up
__device__ __forceinline__ bool chunk_idle(const PagedSeqs& s, const PagedAttnArgs& a) {
  if (!a.fronts_only || s.share[2 * s.B] != 0) return false;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_units = 0;
  if (threadIdx.x == 0) pdl_wait();  // (the kernels behind this one need what the kernels ahead of it wrote)
  return true;
}
// what the chunk kernels make of index b: a chunk's sequence, a group's front (at its first sequence), or nothing
__device__ __forceinline__ bool chunk_seq(const PagedSeqs& s, const PagedAttnArgs& a, int b, PagedSeq& q, int* status) {
  q = paged_seq(s, b, status);
  const int end = s.share ? s.share[s.B + b] : 0;
  if (end == 0) return chunk_class(q, a);
  q.nq = s.cu[end] - q.row0;
  q.cap = q.skip * PG_TILE;
  q.len = q.cap + q.nq;
  return true;
}

// page of the `rows` slots from j on, or one past the last page (the copy then brings zeros) where no row sees any of them
__device__ __forceinline__ int chunk_page(const PagedSeqs& s, const int32_t* pages, int j, int rows, int lo, int hi, int* status) {
  if (j >= hi || j + rows <= lo) return s.n_pages;
  const int pg = pages[j >> s.page_log2];
  if (pg >= 0 && pg < s.n_pages) return pg;
  atomicCAS(status, 0, ST_BAD_INDEX);
  return s.n_pages;
}

int paged_chunk_launch(int D, const PagedPool& kp, const PagedPool& vp, const PagedSeqs& s, const PagedAttnArgs& a, const PagedWeightArgs* w, bool early,
                       cudaStream_t st, int dev, int* status);

}  // namespace spinf
