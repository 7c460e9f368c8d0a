// Attention of a chunk of new tokens over the paged K/V cache (sequences with more than 64 query rows per kv head), tcgen05 + TMEM +
// TMA as CTA pairs.
//
// An item is 256 query rows of one kv head: `hp` heads that share it x 256 / hp tokens, the first half of the tokens in one CTA of
// the pair and the second in the other. The pair walks the key tiles some row sees, 128 keys at a time:
//   warp 0     one lane: TMA loads of Q and of this CTA's 64 keys of K
//   warp 10    TMA loads of this CTA's half of V's dimensions (all 128 keys). In a tile with slots that no row of the item sees (a
//              page's end, the front of a window) it waits for the copy and clears those rows: P is 0 there, but 0 * inf is not
//   warp 1     owns tensor memory; the leader's lane issues S = Q K^T (M = 256) into one of two buffers and O += P V with P read from
//              tensor memory; S of tile t + 1 is issued before P V of tile t
//   warps 2-9  two softmax groups of four warps, thread = row, group A the first 64 keys of the tile and B the others; the mask is
//              arithmetic on slots (a row sees the slots up to its own, with a window the last ones), evaluated on boundary tiles only
// What bounds it: the tensor pipe (4 D flops per pair of row and key). The pair is there for K and V: 128 rows alone would need a
// tile of 128 keys from L2 every 2 048 cycles (D 256), 64 bytes per cycle and SM, more than L2 delivers; 256 rows halve that.
//
// A sequence's work, the (item, key tile) pairs in order, is dealt out in equal contiguous units, one per CTA pair of the GPU
// (fewer for little work): the causal triangle, ragged tails and few items of many tiles balance by themselves. An item cut by
// a unit's border leaves partial rows (maximum, sum, O in fp32), which the join adds in order. The cut depends on the sequence's own
// lengths only, so its results do not depend on the rest of the call.
#include "paged_attn.cuh"

#include <atomic>

namespace spinf {

static constexpr int CH_KH = 64;
static constexpr float CH_RESCALE = 24.f;  // log2 units: the reference maximum moves when a row's maximum grew by more
static constexpr int CHUNK_THREADS = 352;

template <int D>
struct ChunkSmem {
  static constexpr int SLABS = D / 64;
  static constexpr int Q_BYTES = SLABS * 128 * 128;
  static constexpr int KV = SLABS * CH_KH * 128;  // one stage: 64 keys of K, or 128 keys of half of V's dimensions
  static constexpr int NS = D == 256 ? 2 : 4;
  static constexpr int K_OFF = Q_BYTES;
  static constexpr int V_OFF = K_OFF + NS * KV;
  static constexpr int BAR_OFF = V_OFF + NS * KV;
  static constexpr int XCHG_OFF = BAR_OFF + 512;
  static constexpr int PRE_OFF = XCHG_OFF + 3 * 2 * 128 * 4;
  static constexpr int TOTAL = PRE_OFF + (PG_MAX_SEQS + 2) * 4 + 1024;
  static constexpr int TMEM_COLS = 512;  // S: 2 x 128 columns, O: D columns from 256
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
  int g, h0, tok0;     // kv head, first query head, first token of the pair
  int ta, tb;          // key tiles
  int lo, hi;          // slots some row of the item sees
  int64_t part;        // first row of the partial result (256 rows), or -1: the segment is the whole item
};

// walks the segments of a unit; every role of both CTAs walks the same
struct ChunkWalk {
  PagedSeq q;
  ChunkCut c;
  int b, it;
  int64_t w, w_end;  // (item, tile) pairs of the unit still to do
  int tt, nt, t0;    // token tile, its key tiles, the first of them
  int64_t w_tt;      // first pair of the token tile
  bool first;

  __device__ __forceinline__ void start(const PagedSeqs& s, const PagedAttnArgs& a, const int* pre, int it, int* status) {
    b = paged_find(pre, s.B, it);
    q = paged_seq(s, b, status);
    c = chunk_cut(q, a);
    this->it = it;
    const int u = it - pre[b];
    w = c.begin(u);
    w_end = c.begin(u + 1);
    first = true;
    tt = -1, w_tt = 0, nt = 0;
    advance(a);
  }
  // to the token tile that holds pair w
  __device__ __forceinline__ void advance(const PagedAttnArgs& a) {
    while (w >= w_tt + static_cast<int64_t>(nt) * c.per_tt) {
      w_tt += static_cast<int64_t>(nt) * c.per_tt;
      ++tt;
      if (tt >= c.ntt) return;
      c.tiles(q, a, tt, t0, nt);
    }
  }
  __device__ __forceinline__ bool next(const PagedAttnArgs& a, ChunkSeg& g) {
    if (w >= w_end) return false;
    advance(a);
    const int64_t in = w - w_tt;
    const int item = static_cast<int>(in / nt), off = static_cast<int>(in - static_cast<int64_t>(item) * nt);
    const int64_t left = w_end - w;
    const int len = left < nt - off ? static_cast<int>(left) : nt - off;
    const int sets = a.group / c.hp;
    g.g = item / sets;
    g.h0 = g.g * a.group + (item % sets) * c.hp;
    g.tok0 = tt * c.tok;
    g.ta = t0 + off;
    g.tb = g.ta + len;
    c.slots(q, a, tt, g.lo, g.hi);
    g.part = len == nt ? -1 : (static_cast<int64_t>(it) * 2 + (first ? 0 : 1)) * 256;
    first = false;
    w += len;
    return true;
  }
};

template <int D>
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const PagedSeqs s, const PagedAttnArgs a, int* __restrict__ status) {
  using L = ChunkSmem<D>;
  constexpr int SLABS = L::SLABS, NS = L::NS, V_SLABS = SLABS / 2;
  constexpr uint32_t IDESC_S = make_idesc(FMT_BF16, FMT_BF16, 256, 128, 0, 0);
  constexpr uint32_t IDESC_O = make_idesc(FMT_BF16, FMT_BF16, 256, D, 0, 1);  // B = V, MN-major (head dimensions contiguous)

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;
  uint64_t* k_empty = k_full + NS;
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint64_t* s_full = v_empty + NS;  // 2 buffers
  uint64_t* p_ready = s_full + 2;
  uint64_t* o_done = p_ready + 1;
  uint64_t* o_free = o_done + 1;
  uint64_t* v_edge = o_free + 1;  // copies of a boundary tile, in the CTA's own barrier
  uint32_t* tmem_base_p = reinterpret_cast<uint32_t*>(v_edge + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_p + 1);
  float* xchg = reinterpret_cast<float*>(smem + L::XCHG_OFF);
  int* pre = reinterpret_cast<int*>(smem + L::PRE_OFF);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx wc{abort_flag, status};
  const uint32_t rank = cluster_ctarank();
  const int n_pairs = static_cast<int>(gridDim.x) >> 1, pair = static_cast<int>(blockIdx.x) >> 1;
  pdl_trigger();

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 2);  // one arrival of each CTA's V warp: the copies are queued, or the boundary tile is ready
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1);
    mbar_init(p_ready, 16);  // one arrival per softmax warp of both CTAs
    mbar_init(o_done, 1);
    mbar_init(o_free, 16);
    mbar_init(v_edge, 1);
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
  paged_item_prefix(s.B, pre, CHUNK_THREADS, [&](int b) {
    const PagedSeq q = paged_seq(s, b, status);
    return chunk_class(q, a) ? chunk_cut(q, a).units : 0;
  });
  int total = pre[s.B];
  if (total > a.max_units) {  // rows of q that several sequences claim: more units than n rows can make
    total = a.max_units;
    atomicCAS(status, 0, ST_BAD_INDEX);
  }
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= s.B; b += CHUNK_THREADS) a.unit_pre[b] = pre[b];  // the join's index of the partial rows
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before any remote arrival or peer-signalled copy
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_p;
  const int in_page = (1 << s.page_log2) - 1;

  if (warp == 0) {
    if (lane == 0) {
      const int rows = s.page_log2 < 6 ? 1 << s.page_log2 : CH_KH;  // rows of a K box
      uint32_t cnt = 0, seg_n = 0;
      bool ok = true;
      for (int it = pair; it < total && ok; it += n_pairs) {
        ChunkWalk wk;
        wk.start(s, a, pre, it, status);
        const int32_t* pages = s.table + wk.b * s.table_pitch;
        const int hp = wk.c.hp, qrows = 128 / hp;
        ChunkSeg g;
        while (ok && wk.next(a, g)) {
          if (!mbar_wait(wc, q_empty, (seg_n & 1u) ^ 1u, ST_TIMEOUT_EMPTY)) { ok = false; break; }
          if (rank == 0) mbar_expect_tx(q_full, 2 * L::Q_BYTES);
          const int row = wk.q.row0 + g.tok0 + static_cast<int>(rank) * qrows;
          for (int hh = 0; hh < hp; ++hh)
            for (int x = 0; x < SLABS; ++x)
              tma_load_2d_pair(smem + x * 128 * 128 + hh * qrows * 128, &tmQ, (g.h0 + hh) * D + x * 64, row, map_to_cta(q_full, 0));
          ++seg_n;
          for (int t = g.ta; t < g.tb; ++t, ++cnt) {
            const uint32_t st = cnt % NS;
            if (!mbar_wait(wc, &k_empty[st], ((cnt / NS) & 1u) ^ 1u, ST_TIMEOUT_EMPTY)) { ok = false; break; }
            if (rank == 0) mbar_expect_tx(&k_full[st], 2 * L::KV);
            const uint32_t bar = map_to_cta(&k_full[st], 0);
            const int j0 = t * PG_TILE + static_cast<int>(rank) * CH_KH;
            for (int x = 0; x < CH_KH / rows; ++x) {
              const int pg = chunk_page(s, pages, j0 + x * rows, rows, g.lo, g.hi, status);
              const int at = (j0 + x * rows) & in_page;
              uint8_t* dst = smem + L::K_OFF + st * L::KV + x * rows * 128;
              if (rows == CH_KH)
                tma_load_5d_pair(dst, &tmK, 0, at, 0, g.g, pg, bar);
              else
                for (int y = 0; y < SLABS; ++y) tma_load_5d_pair(dst + y * CH_KH * 128, &tmK, 0, at, y, g.g, pg, bar);
            }
          }
        }
      }
    }
  } else if (warp == 10) {
    const int rows = s.page_log2 < 7 ? 1 << s.page_log2 : PG_TILE;  // rows of a V box
    uint32_t cnt = 0, edges = 0;
    bool ok = true;
    for (int it = pair; it < total && ok; it += n_pairs) {
      ChunkWalk wk;
      wk.start(s, a, pre, it, status);
      const int32_t* pages = s.table + wk.b * s.table_pitch;
      ChunkSeg g;
      while (ok && wk.next(a, g)) {
        for (int t = g.ta; t < g.tb; ++t, ++cnt) {
          const uint32_t st = cnt % NS;
          const bool edge = t * PG_TILE < g.lo || (t + 1) * PG_TILE > g.hi;
          if (lane == 0) {
            ok = mbar_wait(wc, &v_empty[st], ((cnt / NS) & 1u) ^ 1u, ST_TIMEOUT_EMPTY);
            if (ok) {
              if (edge)
                mbar_expect_tx(v_edge, L::KV);
              else if (rank == 0)
                mbar_expect_tx(&v_full[st], 2 * L::KV);
              else
                mbar_arrive_cluster(map_to_cta(&v_full[st], 0));
              const uint32_t bar = map_to_cta(&v_full[st], 0);
              for (int x = 0; x < PG_TILE / rows; ++x) {
                const int j = t * PG_TILE + x * rows;
                const int pg = chunk_page(s, pages, j, rows, g.lo, g.hi, status);
                uint8_t* dst = smem + L::V_OFF + st * L::KV + x * rows * 128;
                for (int y = 0; y < (rows == PG_TILE ? 1 : V_SLABS); ++y) {
                  const int slab = static_cast<int>(rank) * V_SLABS + y;
                  if (edge)
                    tma_load_5d(dst + y * PG_TILE * 128, &tmV, 0, j & in_page, slab, g.g, pg, v_edge);
                  else
                    tma_load_5d_pair(dst + y * PG_TILE * 128, &tmV, 0, j & in_page, slab, g.g, pg, bar);
                }
              }
              if (edge) ok = mbar_wait(wc, v_edge, edges & 1u, ST_TIMEOUT_FULL);
            }
          }
          ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
          if (!ok) break;
          if (edge) {
            ++edges;
            for (int x = lane; x < PG_TILE * V_SLABS * 8; x += 32) {
              const int key = (x >> 3) % PG_TILE, slab = (x >> 3) / PG_TILE, j = t * PG_TILE + key;
              if (j < g.lo || j >= g.hi)
                *reinterpret_cast<uint4*>(smem + L::V_OFF + st * L::KV + slab * PG_TILE * 128 + sw128_offset(key, x & 7)) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_release(map_to_cta(&v_full[st], 0));
          }
        }
      }
    }
    if (*abort_flag && lane == 0)  // a boundary tile's copies complete here, not on the leader's barriers
      for (int spin = 0; spin < 4096 && !mbar_try_wait(v_edge, edges & 1u); ++spin) {}
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t q_addr = smem_u32(smem);
      uint32_t kc = 0, vc = 0, gt = 0, seg_n = 0;
      bool ok = true;
      auto issue_s = [&](uint32_t g) -> bool {  // S of tile g into buffer g & 1
        const uint32_t st = kc % NS;
        if (!mbar_wait(wc, &k_full[st], (kc / NS) & 1u, ST_TIMEOUT_FULL)) return false;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(smem + L::K_OFF + st * L::KV);
        const uint32_t d_tmem = tmem_base + (g & 1u) * 128;
#pragma unroll
        for (int x = 0; x < SLABS; ++x) {
          const uint64_t ad = make_smem_desc_sw128(q_addr + x * 128 * 128, 16, 1024);
          const uint64_t bd = make_smem_desc_sw128(k_addr + x * CH_KH * 128, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f16_ss_pair(d_tmem, ad + 2 * k, bd + 2 * k, IDESC_S, (x | k) != 0);
        }
        umma_commit_pair_both(&k_empty[st]);
        umma_commit_pair_both(&s_full[g & 1u]);
        ++kc;
        return true;
      };
      for (int it = pair; it < total && ok; it += n_pairs) {
        ChunkWalk wk;
        wk.start(s, a, pre, it, status);
        ChunkSeg g;
        while (ok && wk.next(a, g)) {
          const int n_tiles = g.tb - g.ta;
          if (!mbar_wait(wc, q_full, seg_n & 1u, ST_TIMEOUT_FULL)) { ok = false; break; }
          tc_fence_after();
          if (!issue_s(gt)) { ok = false; break; }
          for (int i = 0; i < n_tiles; ++i) {
            const uint32_t gi = gt + i;
            if (i + 1 < n_tiles) {
              if (!issue_s(gi + 1)) { ok = false; break; }  // buffer (gi + 1) & 1 last held P of tile gi - 1, whose P V was issued before
            } else {
              umma_commit_pair_both(q_empty);
            }
            if (!mbar_wait(wc, p_ready, gi & 1u, ST_TIMEOUT_OTHER)) { ok = false; break; }
            if (i == 0 && seg_n > 0 && !mbar_wait(wc, o_free, (seg_n - 1) & 1u, ST_TIMEOUT_OTHER)) { ok = false; break; }
            const uint32_t st = vc % NS;
            if (!mbar_wait(wc, &v_full[st], (vc / NS) & 1u, ST_TIMEOUT_FULL)) { ok = false; break; }
            tc_fence_after();
            const uint32_t v_addr = smem_u32(smem + L::V_OFF + st * L::KV);
            const uint64_t vd = make_smem_desc_sw128(v_addr, PG_TILE * 128, 1024);
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const uint32_t p_tmem = tmem_base + (gi & 1u) * 128 + hh * CH_KH;  // packed bf16 P: 16 keys per 8 columns
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16_ts_pair(tmem_base + L::O_COL, p_tmem + 8 * k, vd + 128 * (4 * hh + k), IDESC_O, (i | hh | k) != 0);
            }
            umma_commit_pair_both(&v_empty[st]);
            umma_commit_pair_both(o_done);
            ++vc;
          }
          gt += n_tiles;
          ++seg_n;
        }
      }
    }
  } else {
    // softmax warps 2..9
    const int wg = (warp - 2) >> 2;
    const int qd = warp & 3;  // TMEM lane quarter of this warp
    const int row = qd * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(qd * 32) << 16;
    uint32_t gt = 0;
    bool alive = true;
    for (int it = pair; it < total && alive; it += n_pairs) {
      ChunkWalk wk;
      wk.start(s, a, pre, it, status);
      const int hp = wk.c.hp, qrows = 128 / hp;
      const int base = wk.q.len - wk.q.nq;
      ChunkSeg g;
      while (alive && wk.next(a, g)) {
        const int n_tiles = g.tb - g.ta;
        const int head = g.h0 + row / qrows;
        const int tok_first = g.tok0 + static_cast<int>(rank) * qrows, tok = tok_first + row % qrows;
        const int hi = base + tok, lo = a.window > 0 ? hi - a.window + 1 : 0;  // slots the row sees
        const int hi_min = base + tok_first, lo_max = a.window > 0 ? hi_min + qrows - a.window : 0;
        float m_ref = -INFINITY, l_run = 0.f;
        for (int i = 0; i < n_tiles; ++i) {
          const uint32_t gi = gt + i;
          const int jb = (g.ta + i) * PG_TILE + wg * CH_KH;
          bool got = mbar_wait(wc, &s_full[gi & 1u], (gi >> 1) & 1u, ST_TIMEOUT_TMEM);
          float sc[CH_KH];
          float mx = -INFINITY;
          const uint32_t s_tmem = tmem_base + lane_off + (gi & 1u) * 128 + wg * CH_KH;
          if (__all_sync(0xffffffffu, got)) {
            tc_fence_after();
            uint32_t v0[32], v1[32];
            tmem_ld_x32(s_tmem, v0);
            tmem_ld_x32(s_tmem + 32, v1);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) sc[c] = __uint_as_float(v0[c]), sc[32 + c] = __uint_as_float(v1[c]);
            if (jb + CH_KH - 1 > hi_min || jb < lo_max) {
              uint64_t bits = hi < jb ? 0ull : hi - jb >= 63 ? ~0ull : (2ull << (hi - jb)) - 1ull;
              if (lo > jb) bits &= lo - jb > 63 ? 0ull : ~0ull << (lo - jb);
              const uint32_t b_lo = static_cast<uint32_t>(bits), b_hi = static_cast<uint32_t>(bits >> 32);
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                sc[c] = (b_lo & (1u << c)) ? sc[c] : -INFINITY;
                sc[32 + c] = (b_hi & (1u << c)) ? sc[32 + c] : -INFINITY;
              }
            }
#pragma unroll
            for (int c = 0; c < CH_KH; ++c) mx = fmaxf(mx, sc[c]);
          } else {
            got = false;
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
          const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
          float sum0 = 0.f, sum1 = 0.f;
          uint32_t pk[CH_KH / 2];
#pragma unroll
          for (int c = 0; c < CH_KH / 2; ++c) {
            const float p0 = fast_exp2(fmaf(sc[2 * c], a.scale_log2, neg_m)), p1 = fast_exp2(fmaf(sc[2 * c + 1], a.scale_log2, neg_m));
            sum0 += p0;
            sum1 += p1;
            pk[c] = pack_bf16x2(p0, p1);
          }
          l_run = l_run * alpha + (sum0 + sum1);
          if (i > 0) {
            const bool done = mbar_wait(wc, o_done, (gi - 1) & 1u, ST_TIMEOUT_TMEM);
            if (__any_sync(0xffffffffu, alpha != 1.f) && __all_sync(0xffffffffu, done)) {
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 64; ++c) {
                uint32_t o[32];
                const uint32_t o_tmem = tmem_base + lane_off + L::O_COL + wg * (D / 2) + c * 32;
                tmem_ld_x32(o_tmem, o);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                tmem_st_x32(o_tmem, o);
              }
            }
          }
          __syncwarp();
          tmem_st_x32(s_tmem, pk);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_to_cta(p_ready, 0));
        }
        if (!alive) break;
        gt += n_tiles;

        // end of the segment: O of this group's half of the columns
        float* xq = xchg + 2 * 256;
        xq[wg * 128 + row] = l_run;
        const bool got = mbar_wait(wc, o_done, (gt - 1) & 1u, ST_TIMEOUT_TMEM);
        if (!bar_red_and(1 + qd, 64, got)) { alive = false; break; }
        tc_fence_after();
        const float l = l_run + xq[(wg ^ 1) * 128 + row];
        const bool live = tok < wk.q.nq;
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a row that sees nothing: 0; a NaN sum stays NaN
        __nv_bfloat16* dst = a.out + static_cast<int64_t>(wk.q.row0 + tok) * a.out_pitch + static_cast<int64_t>(head) * D + wg * (D / 2);
        const int64_t prow = g.part + static_cast<int64_t>(rank) * 128 + row;
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld_x32(tmem_base + lane_off + L::O_COL + wg * (D / 2) + c * 32, o);
          tmem_wait_ld();
          if (c == D / 64 - 1) {  // O is in registers: the next segment's first P V may overwrite it
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(o_free, 0));
          }
          if (!live) continue;
          if (g.part < 0) {
            uint32_t wv[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) wv[x] = pack_bf16x2(__uint_as_float(o[2 * x]) * inv, __uint_as_float(o[2 * x + 1]) * inv);
            uint4* to = reinterpret_cast<uint4*>(dst + c * 32);
#pragma unroll
            for (int x = 0; x < 4; ++x) to[x] = make_uint4(wv[4 * x], wv[4 * x + 1], wv[4 * x + 2], wv[4 * x + 3]);
          } else {
            uint4* to = reinterpret_cast<uint4*>(a.chunk_o + prow * D + wg * (D / 2) + c * 32);
#pragma unroll
            for (int x = 0; x < 8; ++x) to[x] = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          }
        }
        if (live && wg == 0) {
          if (g.part >= 0)
            a.chunk_ml[prow] = make_float2(m_ref, l);
          else if (a.lse)
            a.lse[static_cast<int64_t>(wk.q.row0 + tok) * a.H + head] = m_ref + log2f(l);
        }
      }
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

// ---------------------------------------------------------------- join of the cut items
// one warp per (row, head); the pieces of its item are added in the order of the units
template <int D>
__global__ void __launch_bounds__(256) paged_chunk_join_kernel(const PagedSeqs s, const PagedAttnArgs a, int* __restrict__ status) {
  pdl_trigger();
  pdl_wait();
  constexpr int V = D / 128;  // float4 per lane
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedSeq q = paged_seq(s, b, status);
  if (!chunk_class(q, a)) return;
  const ChunkCut c = chunk_cut(q, a);
  if (c.units == 1 || a.unit_pre[b + 1] > a.max_units) return;
  // a CTA takes 8 rows (token, head) at a time, all of one token tile and one head where there are many tokens
  int64_t w_tt = 0;
  int tt = 0, t0 = 0, nt = 0;
  c.tiles(q, a, 0, t0, nt);
  const int64_t all = static_cast<int64_t>(q.nq) * a.H;
  for (int64_t x = blockIdx.x * 8 + warp; x < all; x += gridDim.x * 8) {
    const int tok = static_cast<int>(x / a.H), head = static_cast<int>(x % a.H);
    while (tt < tok / c.tok) {
      w_tt += static_cast<int64_t>(nt) * c.per_tt;
      ++tt;
      c.tiles(q, a, tt, t0, nt);
    }
    const int g = head / a.group, hh = head % a.group, sets = a.group / c.hp;
    const int64_t w0 = w_tt + static_cast<int64_t>(g * sets + hh / c.hp) * nt;
    const int u0 = c.unit_of(w0), u1 = c.unit_of(w0 + nt - 1);
    if (u0 == u1) continue;  // whole in one unit: already written
    const int in_tile = tok - tt * c.tok, qrows = 128 / c.hp;
    const int row = (in_tile / qrows) * 128 + (hh % c.hp) * qrows + in_tile % qrows;
    float m = -INFINITY, l = 0.f;
    auto slot = [&](int u) {  // the piece is the unit's first segment unless the item starts inside the unit
      return ((a.unit_pre[b] + static_cast<int64_t>(u)) * 2 + (c.begin(u) < w0 ? 1 : 0)) * 256 + row;
    };
    for (int u = u0; u <= u1; ++u) m = fmaxf(m, a.chunk_ml[slot(u)].x);
    const float neg_m = m == -INFINITY ? 0.f : -m;
    float4 acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int u = u0; u <= u1; ++u) {
      const int64_t at = slot(u);
      const float2 ml = a.chunk_ml[at];
      const float f = fast_exp2(ml.x + neg_m);
      l = fmaf(f, ml.y, l);
      const float4* src = reinterpret_cast<const float4*>(a.chunk_o + at * D);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float4 z = src[v * 32 + lane];
        acc[v].x = fmaf(f, z.x, acc[v].x), acc[v].y = fmaf(f, z.y, acc[v].y), acc[v].z = fmaf(f, z.z, acc[v].z), acc[v].w = fmaf(f, z.w, acc[v].w);
      }
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    __nv_bfloat16* dst = a.out + (q.row0 + tok) * a.out_pitch + static_cast<int64_t>(head) * D;
#pragma unroll
    for (int v = 0; v < V; ++v)
      *reinterpret_cast<uint2*>(dst + (v * 32 + lane) * 4) =
          make_uint2(pack_bf16x2(acc[v].x * inv, acc[v].y * inv), pack_bf16x2(acc[v].z * inv, acc[v].w * inv));
    if (a.lse && lane == 0) a.lse[static_cast<int64_t>(q.row0 + tok) * a.H + head] = m + log2f(l);
  }
}

template <int D>
static int launch_chunk(const PagedPool& kp, const PagedPool& vp, const PagedSeqs& s, const PagedAttnArgs& a, int64_t max_q, cudaStream_t st, int dev,
                        int* status) {
  using L = ChunkSmem<D>;
  CUtensorMap tmQ, tmK, tmV;
  const int hp = chunk_heads(a.group);
  int r;
  const uint32_t krows = kp.page < CH_KH ? static_cast<uint32_t>(kp.page) : static_cast<uint32_t>(CH_KH);
  const uint32_t vrows = kp.page < PG_TILE ? static_cast<uint32_t>(kp.page) : static_cast<uint32_t>(PG_TILE);
  if ((r = make_tmap_2d(&tmQ, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.q, s.n, static_cast<uint64_t>(a.H) * D, a.q_pitch * 2, 64, 128 / hp))) return r;
  if ((r = make_tmap_pages(&tmK, kp, krows, krows == CH_KH ? D / 64 : 1))) return r;
  if ((r = make_tmap_pages(&tmV, vp, vrows, vrows == PG_TILE ? D / 128 : 1))) return r;
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    SPINF_CUDA_OK(cudaFuncSetAttribute(paged_chunk_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL));
    attr_set[dev].store(true, std::memory_order_release);
  }
  SPINF_CUDA_OK(launch_after(paged_chunk_kernel<D>, dim3(static_cast<unsigned>(sm_count() / 2 * 2)), dim3(CHUNK_THREADS), st, L::TOTAL, 2, tmQ, tmK, tmV, s, a,
                             status));
  int64_t gx = (max_q * a.H + 7) / 8;
  if (gx > 2048) gx = 2048;
  SPINF_CUDA_OK(launch_after(paged_chunk_join_kernel<D>, dim3(static_cast<unsigned>(gx), s.B), dim3(256), st, 0, 1, s, a, status));
  return 0;
}

int paged_chunk_launch(int D, const PagedPool& kp, const PagedPool& vp, const PagedSeqs& s, const PagedAttnArgs& a, int64_t max_q, cudaStream_t st, int dev,
                       int* status) {
  return D == 256 ? launch_chunk<256>(kp, vp, s, a, max_q, st, dev, status) : launch_chunk<128>(kp, vp, s, a, max_q, st, dev, status);
}

}  // namespace spinf
