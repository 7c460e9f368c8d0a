// Attention of new tokens over the paged K/V cache: out = softmax(scale q K^T) V over the slots a row sees. Here: the sequences with few
// rows per key / value head (rows = new tokens x heads that share it), and the call's C entry points; paged_chunk.cu has the others.
//
//   paged_step_kernel    at most 16 rows: a decoding step
//   paged_rows_kernel    up to 32 rows per head set: a question branch, a short chunk
//   paged_join_kernel    joins the splits of a sequence: out = sum_c e^(m_c - m) O_c / sum_c e^(m_c - m) l_c
//   paged_weight_kernel  adds each slot's attention weight, the sum over rows and heads of p, from the scores the first two kept
//
// Both attention kernels: persistent CTAs, one per SM; an item is (sequence, 64-row tile, kv head, split of the keys). A producer warp
// brings K and V pages in with TMA, 64 keys a stage, into one ring that runs ahead across items; the others compute with warp-level
// products (with the rows of q along M a 128-row tensor-core tile would be 8 to 16 times empty; with the keys there, as the weights of
// chunks have them, it was not built) and a running maximum and sum in fp32. P is rounded to bf16 for
// the product (its operands are 16 bit), which adds about what rounding the output to bf16 adds; the sum takes p unrounded.
//
// paged_step_kernel: each warp takes 16 keys against all rows and keeps a maximum, a sum and an output of its own, so that nothing but
// the ring's barriers stands between a key's arrival and its use; the warps' shares are joined once per item. (With a shared maximum,
// as in the rows kernel, 64 sequences of up to 8 192 tokens took 714 us, so 394 to 400.) S^T = K Q^T with the keys as rows: P^T is turned into
// the second product's operand between lanes, without shared memory. Bound by HBM: 64 ragged steps (32 / 16 heads of 128) 394 us, 6.2
// TB/s of K and V; 131 072 slots (24 / 4 heads of 256) 90 us, 6.0 TB/s; a few short sequences by latency: 4 x 1 501 tokens 19 us, of
// which about 7 are the launches of the kernel and the join. Pages of 64 tokens and more are one copy a stage; of 32 tokens two (6.2
// TB/s instead of 6.5), of 16 four (4.8 TB/s).
//
// paged_rows_kernel: S: each warp takes 16 keys of a 128-key tile against all rows. The row maxima are exchanged through shared memory,
// P goes to shared memory as bf16, and for P V each warp takes an eighth of the head dimensions over all 128 keys, so the output needs
// no exchange and K and V are read from shared memory once. Bound by the warp-level products (one m16n8k16 takes a scheduler about 13
// cycles: 24 rows padded to 32 and D 256 make a tile 5 900 cycles, and an item costs about 4 000 more): 56 branches of 12 tokens over
// 2 012 (16 / 8 heads of 256) 224 us.
//
//   paged_share_kernel   finds neighbouring sequences that begin with the same pages (branches of one content). Their common front is then
//                        read once for all of their rows, by the chunk kernels; the kernels here begin behind it: the 56 branches 100 us
//                        (looking 6, few-row part 39, front 40, joins 13), 12 tokens over 16 384 each 1 500 -> 293 us.
#include "paged_attn.cuh"

#include <atomic>

namespace spinf {

static constexpr int PLAN = 32;          // items planned at a time, one per lane of the producer warp
static constexpr int ROWS_THREADS = 288;  // eight warps and the producer

template <int D>
struct RowsSmem {
  static constexpr int SLABS = D / 64;
  static constexpr int STAGE = 64 * D * 2;  // 64 keys of K or V
  static constexpr int NST = D == 256 ? 5 : 10;
  static constexpr int Q_PITCH = D * 2 + 16;  // a row of q; the 16 bytes spread the rows over the banks
  static constexpr int Q_SLOT = RT * Q_PITCH;
  static constexpr int P_OFF = NST * STAGE;
  static constexpr int Q_OFF = P_OFF + RT * PG_TILE * 2;
  static constexpr int RED_OFF = Q_OFF + Q_SLOT;  // [64][8] floats, twice: row maxima, row sums
  static constexpr int ITEM_OFF = RED_OFF + 2 * RT * 8 * 4;
  static constexpr int PRE_OFF = ITEM_OFF + (1 + PLAN) * 64;
  static constexpr int BAR_OFF = PRE_OFF + (PG_MAX_SEQS + 2) * 4;
  static constexpr int TOTAL = BAR_OFF + (2 * NST + 2) * 8 + 16 + 1024;
};
static_assert(RowsSmem<256>::TOTAL <= 232448 && RowsSmem<128>::TOTAL <= 232448, "shared memory of a CTA");
static_assert(RowsSmem<256>::PRE_OFF % 8 == 0 && RowsSmem<256>::BAR_OFF % 8 == 0 && RowsSmem<128>::BAR_OFF % 8 == 0, "alignment");

// what the consumers need of an item; the producer writes it beside the rows of q
struct alignas(4) KeyItem {
  int b, g, split, splits;
  int row0, nq, base;  // first row of q, rows of the sequence, slot of the first
  int r0, rows;        // rows of the item among the sequence's rows of the head (token * group + head in group)
  int lo, hi;          // slots that some row of the item sees
  int u0, u1;          // 64-key units
};

template <bool STEP>
__device__ __forceinline__ int key_items(const PagedSeqs& s, const PagedAttnArgs& a, int b, int* status) {
  const PagedSeq q = paged_seq(s, b, status);
  if (!(STEP ? step_class(q, a) : rows_class(q, a))) return 0;
  const PagedCut c = STEP ? step_cut(q, a) : rows_cut(q, a);
  return a.h * c.row_tiles * c.splits;
}
template <bool STEP>
__device__ __forceinline__ KeyItem key_item(const PagedSeqs& s, const PagedAttnArgs& a, const int* pre, int it, int* status) {
  KeyItem w;
  w.b = paged_find(pre, s.B, it);
  const PagedSeq q = paged_seq(s, w.b, status);
  const PagedCut c = STEP ? step_cut(q, a) : rows_cut(q, a);
  int x = it - pre[w.b];
  w.r0 = STEP ? 0 : x % c.row_tiles * RT;
  if (!STEP) x /= c.row_tiles;
  w.g = x % a.h;
  w.split = x / a.h;
  w.splits = c.splits + (q.skip ? 1 : 0);  // (what the sequence shares with others counts as a split: the item's result is a part)
  w.row0 = q.row0, w.nq = q.nq, w.base = q.len - q.nq;
  const int all = q.nq * a.group;
  w.rows = STEP || all - w.r0 < RT ? all - w.r0 : RT;
  const int first = w.base + w.r0 / a.group, last = w.base + (w.r0 + w.rows - 1) / a.group;
  w.lo = a.window > 0 && first - a.window + 1 > 0 ? first - a.window + 1 : 0;
  w.hi = last + 1 > 0 ? last + 1 : 0;
  const int s0 = c.t_lo + w.split * c.tiles_per_split, s1 = s0 + c.tiles_per_split < c.t_hi ? s0 + c.tiles_per_split : c.t_hi;
  const int e0 = w.lo / PG_TILE, e1 = (w.hi + PG_TILE - 1) / PG_TILE;
  w.u0 = 2 * (s0 > e0 ? s0 : e0);
  w.u1 = 2 * (s1 < e1 ? s1 : e1);
  if (STEP && w.u1 * 64 >= w.hi + 64) w.u1 -= 1;  // units one by one: the last tile's second half may lie behind the last slot
  if (w.u1 < w.u0) w.u1 = w.u0;
  return w;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// The producer warp of both few-row kernels. Items are planned 32 at a time, one per lane, and an item's page indexes are fetched by
// the lanes together, the next item's while this one is copied, so that no step of the copy loop waits for a load of its own. Order of
// the stages: K and V of a unit in turn (STEP), or the two K units of a 128-key tile and then its two V units. One warp has to keep up
// with the SM's share of HBM (a unit of 32 KB every 1 400 cycles at D 128), so the loop is written for few instructions: ring position
// and phase are counted along, and units that lie inside the visible slots (all but the first and last) skip the box tests.
template <int D, bool STEP, int NST, int STAGE, int Q_PITCH, int Q_SLOT, int NQ>
struct KeyProducer {
  const PagedSeqs& s;
  const PagedAttnArgs& a;
  const CUtensorMap* tmK;
  const CUtensorMap* tmV;
  uint8_t* ring;
  uint64_t* full;
  uint64_t* empty;
  const WaitCtx& wc;
  int* status;
  int br, in_page;
  uint32_t st, ph, cnt;  // ring position, its phase, stages queued
  static constexpr int UNITS = STEP ? 1 : 2;

  __device__ __forceinline__ bool wanted(const KeyItem& w, int j) const {  // some row sees the box at slot j
    return j < w.u1 * 64 && j < w.hi && j + (1 << br) > w.lo;
  }
  // table entry of box x of an item (boxes of 2^br slots from its first unit on). Nothing looks at it here: the first look waits for it
  __device__ __forceinline__ int entry(const KeyItem& w, int x) const {
    const int j = (w.u0 * 64) + (x << br);
    return wanted(w, j) ? s.table[w.b * s.table_pitch + (j >> s.page_log2)] : 0;
  }
  template <int BOXES>  // of a unit
  __device__ __forceinline__ bool copy(const KeyItem& w, int pages, int lane) {
    constexpr int ROWS = 64 / BOXES;
    int x = 0;
#pragma unroll 1
    for (int u = w.u0; u < w.u1; u += UNITS, x += UNITS * BOXES) {
      if (x && (x & 31) == 0) pages = entry(w, x + lane);
      int pg[UNITS * BOXES], bytes[UNITS];
      bool all = u * 64 >= w.lo && (u + UNITS) * 64 <= w.hi;
#pragma unroll
      for (int y = 0; y < UNITS * BOXES; ++y) {
        pg[y] = __shfl_sync(0xffffffffu, pages, (x + y) & 31);
        all = all && static_cast<unsigned>(pg[y]) < static_cast<unsigned>(s.n_pages);
      }
#pragma unroll
      for (int v = 0; v < UNITS; ++v) bytes[v] = 64 * D * 2;
      if (!all) {  // boxes that no row sees stay as they are (masked for K, cleared for V)
#pragma unroll
        for (int y = 0; y < UNITS * BOXES; ++y) {
          const bool want = wanted(w, u * 64 + y * ROWS), good = static_cast<unsigned>(pg[y]) < static_cast<unsigned>(s.n_pages);
          if (!want) {
            pg[y] = -1;
            bytes[y / BOXES] -= ROWS * D * 2;
          } else if (!good) {  // one past the last page: the copy brings zeros
            pg[y] = s.n_pages;
            if (lane == 0) atomicCAS(status, 0, ST_BAD_INDEX);
          }
        }
      }
#pragma unroll
      for (int part = 0; part < 2 * UNITS; ++part) {
        if (!__all_sync(0xffffffffu, mbar_wait(wc, &empty[st], ph ^ 1u, ST_TIMEOUT_EMPTY))) return false;
        if (lane == 0) {
          mbar_expect_tx(&full[st], bytes[part % UNITS]);
#pragma unroll
          for (int y = 0; y < BOXES; ++y)
            if (pg[(part % UNITS) * BOXES + y] >= 0)
              tma_load_5d(ring + st * STAGE + y * (ROWS * D * 2), part < UNITS ? tmK : tmV, 0, ((u + part % UNITS) * 64 + y * ROWS) & in_page, 0, w.g,
                          pg[(part % UNITS) * BOXES + y], &full[st]);
        }
        if (++st == NST) st = 0, ph ^= 1u;
        ++cnt;
      }
    }
    return true;
  }
  __device__ __forceinline__ void run(const int* pre, int total, uint8_t* q_slots, KeyItem* items, KeyItem* plan, uint64_t* q_full, uint64_t* q_empty) {
    const int lane = threadIdx.x & 31;
    uint32_t item_n = 0;
    bool ok = true;
    for (int k0 = 0; ok && static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(k0) * gridDim.x < total; k0 += PLAN) {
      const int64_t mine = static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(k0 + lane) * gridDim.x;
      __syncwarp();
      if (mine < total) plan[lane] = key_item<STEP>(s, a, pre, static_cast<int>(mine), status);
      const int n_plan = __popc(__ballot_sync(0xffffffffu, mine < total));
      __syncwarp();
      int pages_next = entry(plan[0], lane);
      for (int k = 0; k < n_plan; ++k, ++item_n) {
        const KeyItem w = plan[k];
        const int pages = pages_next;
        if (k + 1 < n_plan) pages_next = entry(plan[k + 1], lane);
        const uint32_t qs = item_n % NQ;
        ok = __all_sync(0xffffffffu, mbar_wait(wc, &q_empty[qs], ((item_n / NQ) & 1u) ^ 1u, ST_TIMEOUT_EMPTY));
        if (!ok) break;
        if (lane == 0) {
          items[qs] = w;
          mbar_expect_tx(&q_full[qs], w.rows * D * 2);  // (an arrival: releases the item's numbers to the consumers as well)
        }
        __syncwarp();
        for (int r = lane; r < w.rows; r += 32) {
          const int rr = w.r0 + r;
          bulk_load(q_slots + qs * Q_SLOT + r * Q_PITCH, a.q + (w.row0 + rr / a.group) * a.q_pitch + static_cast<int64_t>(w.g * a.group + rr % a.group) * D,
                    D * 2, &q_full[qs]);
        }
        ok = br == 6 ? copy<1>(w, pages, lane) : br == 5 ? copy<2>(w, pages, lane) : copy<4>(w, pages, lane);
        if (!ok) break;
      }
    }
    if (*wc.abort_flag && lane == 0) {  // bounded wait for copies that may still be in flight
      for (uint32_t c = cnt > static_cast<uint32_t>(NST) ? cnt - NST : 0; c < cnt; ++c)
        for (int spin = 0; spin < 4096 && !mbar_try_wait(&full[c % NST], (c / NST) & 1u); ++spin) {}
      for (uint32_t c = item_n > static_cast<uint32_t>(NQ) ? item_n - NQ : 0u; c <= item_n; ++c)
        for (int spin = 0; spin < 4096 && !mbar_try_wait(&q_full[c % NQ], (c / NQ) & 1u); ++spin) {}
    }
  }
};

// D (16 x 8, fp32) += A (16 x 16, bf16, row) B (16 x 8, bf16, col). Not volatile: the fragment loads are, so the compiler may put the
// loads of the next steps between a load and its product; with both volatile every step waited out its own loads.
__device__ __forceinline__ void mma_free(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// byte offset of (key, 16-byte chunk of its row) in a stage: boxes of 2^br rows x all slabs, 128-byte swizzled
template <int D>
__device__ __forceinline__ uint32_t stage_offset(int key, int chunk, int br) {
  const int box = key >> br, row = key & ((1 << br) - 1);
  return box * (D * 2 << br) + ((chunk >> 3) * 128 << br) + sw128_offset(row, chunk & 7);
}

template <int D, int MT>
__device__ __forceinline__ bool rows_work(const PagedAttnArgs& a, const KeyItem& w, uint8_t* smem, uint64_t* full, uint64_t* empty, uint64_t* q_empty,
                                          uint32_t& cnt, const WaitCtx& wc, int br) {
  using L = RowsSmem<D>;
  constexpr int KS = D / 16;       // 16-dimension steps of S
  constexpr int DW = D / 8;        // head dimensions a warp takes in P V
  constexpr int NT = DW / 8;       // 8-column tiles of them
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3;
  float* red_m = reinterpret_cast<float*>(smem + L::RED_OFF);
  float* red_l = red_m + RT * 8;
  const uint32_t q_base = smem_u32(smem + L::Q_OFF), p_base = smem_u32(smem + L::P_OFF);
  const int t0 = w.u0 / 2, t1 = w.u1 / 2;

  // this thread's rows: 16 m + lane / 4 and 8 more; the slots each sees
  int lo_r[MT][2], hi_r[MT][2];
  int lo_max = 0, hi_min = 0x7fffffff;
  {
    const int base = w.base;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        int r = m * 16 + (lane >> 2) + 8 * x;
        r = r < w.rows ? r : w.rows - 1;
        const int slot = base + (w.r0 + r) / a.group;
        hi_r[m][x] = slot;
        lo_r[m][x] = a.window > 0 ? slot - a.window + 1 : 0;
      }
    lo_max = a.window > 0 ? base + (w.r0 + w.rows - 1) / a.group - a.window + 1 : 0;
    hi_min = base + w.r0 / a.group;
  }
  float o[MT][NT][4];
  float m_run[MT][2], l_run[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[m][t][x] = 0.f;
    m_run[m][0] = m_run[m][1] = -INFINITY;
    l_run[m][0] = l_run[m][1] = 0.f;
  }

  for (int t = t0; t < t1; ++t, cnt += 4) {
    // ---- S of this warp's 16 keys
    const int hf = warp >> 2, key0 = (warp & 3) * 16;  // stage of the tile, first key within it
    bool ok = true;
    {
      const uint32_t c = cnt + hf;
      ok = mbar_wait(wc, &full[c % L::NST], (c / L::NST) & 1u, ST_TIMEOUT_FULL);
    }
    float sc[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int x = 0; x < 4; ++x) sc[m][0][x] = sc[m][1][x] = 0.f;
    if (ok) {
      const uint32_t k_base = smem_u32(smem) + ((cnt + hf) % L::NST) * L::STAGE;
      const int kk = key0 + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t kf[4];
        const uint32_t ka = k_base + stage_offset<D>(kk, ks * 2 + ((lane >> 3) & 1), br);
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(kf[0]), "=r"(kf[1]), "=r"(kf[2]), "=r"(kf[3]) : "r"(ka));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t qf[4];
          const int chunk = ks * 2 + (lane >> 4);
          const uint32_t qa = q_base + (m * 16 + (lane & 15)) * L::Q_PITCH + chunk * 16;
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(qf[0]), "=r"(qf[1]), "=r"(qf[2]), "=r"(qf[3]) : "r"(qa));
          mma_free(sc[m][0], qf, kf[0], kf[1]);
          mma_free(sc[m][1], qf, kf[2], kf[3]);
        }
      }
    }
    __syncwarp();
    if (lane == 0) {  // this warp has read its keys of the two K stages (it used one of them)
      mbar_arrive(&empty[cnt % L::NST]);
      mbar_arrive(&empty[(cnt + 1) % L::NST]);
      if (t == t1 - 1) mbar_arrive(q_empty);  // and q for the last time
    }
    // ---- mask, row maxima
    const int j0 = t * PG_TILE + hf * 64 + key0 + quad * 2;
    const bool masked = (t + 1) * PG_TILE - 1 > hi_min || t * PG_TILE < lo_max;
    float mx[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      mx[m][0] = mx[m][1] = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float v = sc[m][nt][x] * a.scale_log2;
          const int j = j0 + nt * 8 + (x & 1);
          if (masked && (j > hi_r[m][x >> 1] || j < lo_r[m][x >> 1])) v = -INFINITY;
          sc[m][nt][x] = v;
          mx[m][x >> 1] = fmaxf(mx[m][x >> 1], v);
        }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mx[m][x] = fmaxf(mx[m][x], __shfl_xor_sync(0xffffffffu, mx[m][x], 1));
        mx[m][x] = fmaxf(mx[m][x], __shfl_xor_sync(0xffffffffu, mx[m][x], 2));
        if (quad == 0) red_m[(m * 16 + (lane >> 2) + 8 * x) * 8 + warp] = mx[m][x];
      }
    }
    if (a.scores) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = m * 16 + (lane >> 2) + 8 * x;
          if (r < w.rows) {
            const int rr = w.r0 + r;
            float* dst = a.scores + ((static_cast<int64_t>(w.b) * a.tok_cap + rr / a.group) * a.H + w.g * a.group + rr % a.group) * a.score_pitch + j0;
            *reinterpret_cast<float2*>(dst) = make_float2(sc[m][0][2 * x], sc[m][0][2 * x + 1]);
            *reinterpret_cast<float2*>(dst + 8) = make_float2(sc[m][1][2 * x], sc[m][1][2 * x + 1]);
          }
        }
    }
    if (!bar_red_and(1, 256, ok)) return false;
    // ---- new maxima, P
    float alpha[MT][2];
    bool moved = false;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = m * 16 + (lane >> 2) + 8 * x;
        const float4 u = *reinterpret_cast<const float4*>(red_m + r * 8), v = *reinterpret_cast<const float4*>(red_m + r * 8 + 4);
        const float m_new = fmaxf(m_run[m][x], fmaxf(fmaxf(fmaxf(u.x, u.y), fmaxf(u.z, u.w)), fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w))));
        alpha[m][x] = m_new == m_run[m][x] ? 1.f : fast_exp2(m_run[m][x] - m_new);  // (equal covers a row that has seen nothing yet)
        moved |= alpha[m][x] != 1.f;
        m_run[m][x] = m_new;
        const float neg_m = m_new == -INFINITY ? 0.f : -m_new;
        float sum = 0.f;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const float p0 = fast_exp2(sc[m][nt][2 * x] + neg_m), p1 = fast_exp2(sc[m][nt][2 * x + 1] + neg_m);
          sum += p0 + p1;
          const int col = hf * 64 + key0 + nt * 8;  // key of the tile
          const uint32_t off = (col >> 6) * (RT * 128) + sw128_offset(r, (col >> 3) & 7) + quad * 4;
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(p_base + off), "r"(pack_bf16x2(p0, p1)) : "memory");
        }
        l_run[m][x] = l_run[m][x] * alpha[m][x] + sum;
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[m][nt][x] *= alpha[m][x >> 1];
    }
    named_bar_sync(1, 256);
    // ---- O += P V over this warp's head dimensions
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t c = cnt + 2 + half, st = c % L::NST;
      ok = ok && mbar_wait(wc, &full[st], (c / L::NST) & 1u, ST_TIMEOUT_FULL);
      if (ok) {
        const int j_first = t * PG_TILE + half * 64;
        if (j_first < w.lo || j_first + 64 > w.hi) {
          // slots no row of the tile sees may hold anything (or were not copied): p is 0 there, but 0 * inf is not. Each warp clears
          // what it reads.
          for (int x = lane; x < 64 * (DW / 8); x += 32) {
            const int key = x / (DW / 8), ch = warp * (DW / 8) + x % (DW / 8);
            if (j_first + key < w.lo || j_first + key >= w.hi)
              *reinterpret_cast<uint4*>(smem + st * L::STAGE + stage_offset<D>(key, ch, br)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();  // the stage is refilled by the copy engine
          __syncwarp();
        }
        const uint32_t v_base = smem_u32(smem) + st * L::STAGE;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t pf[MT][4];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint32_t pa = p_base + half * (RT * 128) + sw128_offset(m * 16 + (lane & 15), kk * 2 + (lane >> 4));
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(pf[m][0]), "=r"(pf[m][1]), "=r"(pf[m][2]), "=r"(pf[m][3]) : "r"(pa));
          }
          const int key = kk * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            uint32_t vf[4];
            const uint32_t va = v_base + stage_offset<D>(key, warp * (DW / 8) + np * 2 + (lane >> 4), br);
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(vf[0]), "=r"(vf[1]), "=r"(vf[2]), "=r"(vf[3]) : "r"(va));
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              mma_free(o[m][2 * np], pf[m], vf[0], vf[1]);
              mma_free(o[m][2 * np + 1], pf[m], vf[2], vf[3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    if (!ok) *wc.abort_flag = 1;  // the next barrier with a vote ends the CTA's warps together
  }
  if (t1 <= t0 && lane == 0) mbar_arrive(q_empty);
  // ---- row sums over the warps' keys, then the rows out
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float l = l_run[m][x];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (quad == 0) red_l[(m * 16 + (lane >> 2) + 8 * x) * 8 + warp] = l;
    }
  if (!bar_red_and(1, 256, !*wc.abort_flag)) return false;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = m * 16 + (lane >> 2) + 8 * x;
      if (r >= w.rows) continue;
      const float4 u = *reinterpret_cast<const float4*>(red_l + r * 8), v = *reinterpret_cast<const float4*>(red_l + r * 8 + 4);
      const float l = ((u.x + u.y) + (u.z + u.w)) + ((v.x + v.y) + (v.z + v.w));
      const int rr = w.r0 + r, tok = rr / a.group, hd = w.g * a.group + rr % a.group;
      if (w.splits == 1) {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a row that sees nothing: 0; a NaN sum stays NaN
        __nv_bfloat16* dst = a.out + (w.row0 + tok) * a.out_pitch + static_cast<int64_t>(hd) * D + warp * DW + quad * 2;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<uint32_t*>(dst + nt * 8) = pack_bf16x2(o[m][nt][2 * x] * inv, o[m][nt][2 * x + 1] * inv);
        if (a.lse && warp == 0 && quad == 0) a.lse[static_cast<int64_t>(w.row0 + tok) * a.H + hd] = m_run[m][x] + log2f(l);
      } else {
        const int64_t at = w.b * a.seq_parts + (static_cast<int64_t>(w.split) * a.h + w.g) * (w.nq * a.group) + rr;
        float* dst = a.part_o + at * D + warp * DW + quad * 2;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) *reinterpret_cast<float2*>(dst + nt * 8) = make_float2(o[m][nt][2 * x], o[m][nt][2 * x + 1]);
        if (warp == 0 && quad == 0) a.part_ml[at] = make_float2(m_run[m][x], l);
      }
    }
  return true;
}

template <int D>
__global__ void __launch_bounds__(ROWS_THREADS, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PagedSeqs s, const PagedAttnArgs a,
                  int* __restrict__ status) {
  using L = RowsSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  int* pre = reinterpret_cast<int*>(smem + L::PRE_OFF);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* empty = full + L::NST;
  uint64_t* q_full = empty + L::NST;
  uint64_t* q_empty = q_full + 1;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(q_empty + 1);
  const WaitCtx wc{abort_flag, status};
  const int warp = threadIdx.x >> 5;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::NST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 8);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 8);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  paged_item_prefix(s.B, pre, ROWS_THREADS, [&](int b) { return key_items<false>(s, a, b, status); });
  const int total = pre[s.B];
  const int br = s.page_log2 < 6 ? s.page_log2 : 6;  // log2 of a box's rows
  KeyItem* items = reinterpret_cast<KeyItem*>(smem + L::ITEM_OFF);

  if (warp == 8) {
    KeyProducer<D, false, L::NST, L::STAGE, L::Q_PITCH, L::Q_SLOT, 1> p{s, a, &tmK, &tmV, smem, full, empty, wc, status, br, (1 << s.page_log2) - 1, 0, 0, 0};
    p.run(pre, total, smem + L::Q_OFF, items, items + 1, q_full, q_empty);
  } else {
    uint32_t cnt = 0, item_n = 0;
    for (int it = blockIdx.x; it < total; it += gridDim.x, ++item_n) {
      if (!bar_red_and(1, 256, mbar_wait(wc, q_full, item_n & 1u, ST_TIMEOUT_FULL))) break;  // (also: the last item's sums have been read)
      const KeyItem w = items[0];
      bool ok;
      switch ((w.rows + 15) >> 4) {
        case 1: ok = rows_work<D, 1>(a, w, smem, full, empty, q_empty, cnt, wc, br); break;
        case 2: ok = rows_work<D, 2>(a, w, smem, full, empty, q_empty, cnt, wc, br); break;
        case 3: ok = rows_work<D, 3>(a, w, smem, full, empty, q_empty, cnt, wc, br); break;
        default: ok = rows_work<D, 4>(a, w, smem, full, empty, q_empty, cnt, wc, br); break;
      }
      if (!ok) break;
    }
  }
  if (threadIdx.x == 0) pdl_wait();  // the kernels behind this one need what the kernel ahead of it wrote, too
  __syncthreads();
}

// ---------------------------------------------------------------- few rows per kv head (at most 16): a decoding step
// Consumer warps; one more is the producer. D 128: eight in two groups of four that take the 64-key units in turn, a warp 16 keys of
// each; with an even number of units in the ring a stage always belongs to the same group. D 256: a warp's share of the output alone
// is 128 registers (16 rows), so seven (8 warps of 255 registers), which take the units' 16-key pieces in turn.
__host__ __device__ constexpr int step_warps(int D) { return D == 256 ? 7 : 8; }
__host__ __device__ constexpr int step_threads(int D) { return (step_warps(D) + 1) * 32; }

template <int D>
struct StepSmem {
  static constexpr int STAGE = 64 * D * 2;          // 64 keys of K or V
  static constexpr int NST = D == 256 ? 5 : 12;
  static constexpr int Q_PITCH = D * 2 + 16;        // a row of q; the 16 bytes spread the rows over the banks
  static constexpr int Q_SLOT = STEP_ROWS * Q_PITCH;
  static constexpr int SW = step_warps(D);
  static constexpr int MR = 4;                      // rows merged at a time
  static constexpr int Q_OFF = NST * STAGE;
  static constexpr int MERGE_OFF = Q_OFF + 2 * Q_SLOT;
  static constexpr int ML_OFF = MERGE_OFF + SW * MR * D * 4;  // [SW][16] maxima, [SW][16] sums, [16] joined maxima, [16] joined sums
  static constexpr int ITEM_OFF = ML_OFF + (2 * SW + 2) * STEP_ROWS * 4;
  static constexpr int PRE_OFF = ITEM_OFF + (2 + PLAN) * 64;
  static constexpr int BAR_OFF = PRE_OFF + (PG_MAX_SEQS + 2) * 4;
  static constexpr int TOTAL = BAR_OFF + (2 * NST + 4) * 8 + 16 + 1024;
};
static_assert(StepSmem<256>::TOTAL <= 232448 && StepSmem<128>::TOTAL <= 232448, "shared memory of a CTA");
static_assert(StepSmem<256>::BAR_OFF % 8 == 0 && StepSmem<128>::BAR_OFF % 8 == 0 && StepSmem<256>::MERGE_OFF % 16 == 0 &&
                  StepSmem<128>::MERGE_OFF % 16 == 0 && StepSmem<256>::ITEM_OFF % 16 == 0 && StepSmem<128>::ITEM_OFF % 16 == 0, "alignment");

__device__ __forceinline__ void movmatrix_t(uint32_t& d, uint32_t s) {
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(s));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// NT: 8-row tiles of q. A row's arithmetic is the same for either.
template <int D, int NT>
__global__ void __launch_bounds__(step_threads(D), 1)
paged_step_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PagedSeqs s, const PagedAttnArgs a,
                  int* __restrict__ status) {
  using L = StepSmem<D>;
  constexpr int KS = D / 16, SW = L::SW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  int* pre = reinterpret_cast<int*>(smem + L::PRE_OFF);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* empty = full + L::NST;
  uint64_t* q_full = empty + L::NST;
  uint64_t* q_empty = q_full + 2;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(q_empty + 2);
  const WaitCtx wc{abort_flag, status};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (s.share) pdl_wait();  // the groups are the kernel's ahead; all kernels behind this one start after this
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::NST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], D == 256 ? SW : 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], SW);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  paged_item_prefix(s.B, pre, step_threads(D), [&](int b) { return key_items<true>(s, a, b, status); });
  const int total = pre[s.B];
  const int br = s.page_log2 < 6 ? s.page_log2 : 6;  // log2 of a box's rows
  KeyItem* items = reinterpret_cast<KeyItem*>(smem + L::ITEM_OFF);

  if (warp == SW) {
    KeyProducer<D, true, L::NST, L::STAGE, L::Q_PITCH, L::Q_SLOT, 2> p{s, a, &tmK, &tmV, smem, full, empty, wc, status, br, (1 << s.page_log2) - 1, 0, 0, 0};
    p.run(pre, total, smem + L::Q_OFF, items, items + 2, q_full, q_empty);
  } else {
    float* m_w = reinterpret_cast<float*>(smem + L::ML_OFF);  // [SW][16]
    float* l_w = m_w + SW * STEP_ROWS;
    float* m_all = l_w + SW * STEP_ROWS;
    float* l_all = m_all + STEP_ROWS;
    float* merge = reinterpret_cast<float*>(smem + L::MERGE_OFF);
    const uint32_t ring = smem_u32(smem);
    const int c4 = lane & 3, r8 = lane >> 2;
    uint32_t cnt0 = 0, item_n = 0;  // stages before the item, items so far
    for (int it = blockIdx.x; it < total; it += gridDim.x, ++item_n) {
      const uint32_t qs = item_n & 1u;
      bool ok = mbar_wait(wc, &q_full[qs], (item_n >> 1) & 1u, ST_TIMEOUT_FULL);
      ok = __all_sync(0xffffffffu, ok);
      const KeyItem w = items[qs];
      const int rows = w.rows;
      uint32_t qf[NT][KS][2];  // q as the B operand: rows 8 n + lane / 4, dimensions 16 ks + 2 (lane % 4) and 8 more
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int ks = 0; ks < KS; ks += 2) {
          uint32_t r[4];
          ldsm4(r, smem_u32(smem + L::Q_OFF + qs * L::Q_SLOT) + (n * 8 + (lane & 7)) * L::Q_PITCH + ks * 32 + (lane >> 3) * 16);
          qf[n][ks][0] = r[0], qf[n][ks][1] = r[1], qf[n][ks + 1][0] = r[2], qf[n][ks + 1][1] = r[3];
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[qs]);
      if (!ok) {  // the other warps leave at the vote below too: the abort flag is up
        bar_red_and(1, SW * 32, false);
        break;
      }
      // this thread's rows: 8 n + 2 (lane % 4) and the next; the slots each sees
      int hi_r[NT][2], lo_r[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          int r = n * 8 + 2 * c4 + x;
          r = r < rows ? r : rows - 1;
          hi_r[n][x] = w.base + r / a.group;
          lo_r[n][x] = a.window > 0 ? hi_r[n][x] - a.window + 1 : 0;
        }
      const int hi_min = w.base, lo_max = a.window > 0 ? w.hi - a.window : 0;
      float o[KS][NT][4];  // O^T: dimensions 16 i + lane / 4 and 8 more, rows as above
      float m_run[NT][2], l_run[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[i][n][x] = 0.f;
        m_run[n][0] = m_run[n][1] = -INFINITY;
        l_run[n][0] = l_run[n][1] = 0.f;
      }
      // A unit is four pieces of 16 keys. A barrier's parity tells a phase only from its neighbours, so a warp has to wait for every use
      // of every stage it waits for at all. D 128: the groups' stages are their own. D 256: all warps wait for every stage and let it go,
      // also where they have no piece. `me`: the warp's place in the item, which is where its keys are, whatever came before in the ring.
      const int units = w.u1 - w.u0;
      const int me = D == 256 ? warp : ((((warp >> 2) ^ (cnt0 >> 1)) & 1) << 2) + (warp & 3);
      int turn = D == 256 ? warp : warp & 3;  // pieces from the unit's first on to this warp's next
      for (int u = D == 256 ? 0 : me >> 2; u < units && ok; u += D == 256 ? 1 : 2) {
        const uint32_t ck = cnt0 + 2 * u, stk = ck % L::NST, stv = (ck + 1) % L::NST;
        ok = __all_sync(0xffffffffu, mbar_wait(wc, &full[stk], (ck / L::NST) & 1u, ST_TIMEOUT_FULL));
        if (!ok) break;
        const int piece = turn;
        if (D == 256) {
          turn = turn < 4 ? turn + SW - 4 : turn - 4;
          if (piece >= 4) {
            if (lane == 0) mbar_arrive(&empty[stk]);
            ok = __all_sync(0xffffffffu, mbar_wait(wc, &full[stv], ((ck + 1) / L::NST) & 1u, ST_TIMEOUT_FULL));
            if (ok && lane == 0) mbar_arrive(&empty[stv]);
            continue;
          }
        }
        const int key0 = piece * 16, j0 = (w.u0 + u) * 64 + key0;
        float sc[2][NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) sc[0][n][x] = sc[1][n][x] = 0.f;
        {
          const uint32_t k_base = ring + stk * L::STAGE;
          const int key = key0 + (lane & 15);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t kf[4];
            ldsm4(kf, k_base + stage_offset<D>(key, ks * 2 + (lane >> 4), br));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_free(sc[ks & 1][n], kf, qf[n][ks][0], qf[n][ks][1]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stk]);
        const bool masked = j0 + 15 > hi_min || j0 < lo_max;
        uint32_t pf[NT][2];
        bool moved = false;
        float alpha[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float v[4];  // (key, row): (r8, 0) (r8, 1) (r8 + 8, 0) (r8 + 8, 1)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            v[x] = (sc[0][n][x] + sc[1][n][x]) * a.scale_log2;
            const int j = j0 + r8 + (x >> 1) * 8;
            if (masked && (j > hi_r[n][x & 1] || j < lo_r[n][x & 1])) v[x] = -INFINITY;
          }
          if (a.scores) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int r = n * 8 + 2 * c4 + x;
              if (r < rows) {
                float* dst = a.scores + ((static_cast<int64_t>(w.b) * a.tok_cap + r / a.group) * a.H + w.g * a.group + r % a.group) * a.score_pitch + j0 + r8;
                dst[0] = v[x];
                dst[8] = v[2 + x];
              }
            }
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float mx = fmaxf(v[x], v[2 + x]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float m_new = fmaxf(m_run[n][x], mx);
            alpha[n][x] = m_new == m_run[n][x] ? 1.f : fast_exp2(m_run[n][x] - m_new);
            moved |= alpha[n][x] != 1.f;
            m_run[n][x] = m_new;
            const float neg_m = m_new == -INFINITY ? 0.f : -m_new;
            v[x] = fast_exp2(v[x] + neg_m);
            v[2 + x] = fast_exp2(v[2 + x] + neg_m);
            l_run[n][x] = l_run[n][x] * alpha[n][x] + (v[x] + v[2 + x]);
          }
          // P^T (keys x rows) -> the B operand of O^T: 8 x 8 blocks transposed between lanes
          movmatrix_t(pf[n][0], pack_bf16x2(v[0], v[1]));
          movmatrix_t(pf[n][1], pack_bf16x2(v[2], v[3]));
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[i][n][x] *= alpha[n][x & 1];
        }
        ok = __all_sync(0xffffffffu, mbar_wait(wc, &full[stv], ((ck + 1) / L::NST) & 1u, ST_TIMEOUT_FULL));
        if (!ok) break;
        if (j0 < w.lo || j0 + 16 > w.hi) {
          // slots no row sees may hold anything (or were not copied): p is 0 there, but 0 * inf is not
          for (int x = lane; x < 16 * (D / 8); x += 32) {
            const int key = key0 + x / (D / 8);
            const int j = (w.u0 + u) * 64 + key;
            if (j < w.lo || j >= w.hi) *reinterpret_cast<uint4*>(smem + stv * L::STAGE + stage_offset<D>(key, x % (D / 8), br)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();  // the stage is refilled by the copy engine
          __syncwarp();
        }
        {
          const uint32_t v_base = ring + stv * L::STAGE;
          const int key = key0 + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            uint32_t vf[4];
            ldsm4_t(vf, v_base + stage_offset<D>(key, i * 2 + ((lane >> 3) & 1), br));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_free(o[i][n], vf, pf[n][0], pf[n][1]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stv]);
      }
      cnt0 += 2 * (w.u1 > w.u0 ? w.u1 - w.u0 : 0);
      // ---- the warps' shares joined, in the order of their places
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float l = l_run[n][x];
          l += __shfl_xor_sync(0xffffffffu, l, 4);
          l += __shfl_xor_sync(0xffffffffu, l, 8);
          l += __shfl_xor_sync(0xffffffffu, l, 16);
          if (r8 == 0) {
            const int r = n * 8 + 2 * c4 + x;
            m_w[me * STEP_ROWS + r] = m_run[n][x];
            l_w[me * STEP_ROWS + r] = l;
          }
        }
      if (!bar_red_and(1, SW * 32, ok)) break;
      float f[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = n * 8 + 2 * c4 + x;
          float m = -INFINITY, l = 0.f;
#pragma unroll
          for (int y = 0; y < SW; ++y) m = fmaxf(m, m_w[y * STEP_ROWS + r]);
          const float neg_m = m == -INFINITY ? 0.f : -m;
#pragma unroll
          for (int y = 0; y < SW; ++y) l = fmaf(fast_exp2(m_w[y * STEP_ROWS + r] + neg_m), l_w[y * STEP_ROWS + r], l);
          f[n][x] = fast_exp2(m_run[n][x] + neg_m);
          if (warp == 0 && r8 == 0) m_all[r] = m, l_all[r] = l;
        }
      for (int rb = 0; rb < rows; rb += L::MR) {
        if (rb) named_bar_sync(1, SW * 32);  // the rows before these have been read
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r = n * 8 + 2 * c4 + x;
            if (r >= rb && r < rb + L::MR && r < rows) {
              float* dst = merge + (me * L::MR + r - rb) * D + r8;
#pragma unroll
              for (int i = 0; i < KS; ++i) dst[i * 16] = o[i][n][x] * f[n][x], dst[i * 16 + 8] = o[i][n][2 + x] * f[n][x];
            }
          }
        named_bar_sync(1, SW * 32);
        const int n_rows = rows - rb < L::MR ? rows - rb : L::MR;
        for (int x = threadIdx.x; x < n_rows * (D / 4); x += SW * 32) {
          const int r = rb + x / (D / 4), d = (x % (D / 4)) * 4;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int y = 0; y < SW; ++y) {
            const float4 v = *reinterpret_cast<const float4*>(merge + (y * L::MR + r - rb) * D + d);
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
          }
          const int tok = r / a.group, hd = w.g * a.group + r % a.group;
          if (w.splits == 1) {
            const float l = l_all[r], inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a row that sees nothing: 0; a NaN sum stays NaN
            *reinterpret_cast<uint2*>(a.out + (w.row0 + tok) * a.out_pitch + static_cast<int64_t>(hd) * D + d) =
                make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
            if (a.lse && d == 0) a.lse[static_cast<int64_t>(w.row0 + tok) * a.H + hd] = m_all[r] + log2f(l);
          } else {
            const int64_t at = w.b * a.seq_parts + (static_cast<int64_t>(w.split) * a.h + w.g) * rows + r;
            *reinterpret_cast<float4*>(a.part_o + at * D + d) = acc;
            if (d == 0) a.part_ml[at] = make_float2(m_all[r], l_all[r]);
          }
        }
      }
    }
  }
  __syncthreads();
}

// Joins the splits of a (row, head). With few splits a warp takes one; with many the CTA does, its threads in groups of D / 4 that
// share the splits out (a decoding step has few rows and many splits: read one after the other they would be a chain of latencies).
template <int D>
__global__ void __launch_bounds__(256, 4) paged_join_kernel(const PagedSeqs s, const PagedAttnArgs a, int* __restrict__ status) {
  constexpr int V = D / 128;       // float4 per lane of a warp
  constexpr int G = 256 / (D / 4);  // groups of the CTA
  __shared__ float4 part[G][D / 4];
  __shared__ float part_l[G];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedSeq q = paged_seq(s, b, status);
  if (q.nq == 0 || q.skip || chunk_class(q, a)) return;
  const PagedCut c = attn_cut(q, a);
  if (c.splits == 1) return;
  const int all = q.nq * a.group, rows = q.nq * a.H;
  const int64_t step = static_cast<int64_t>(a.h) * all;
  const bool few = c.splits <= 4;
  for (int x = few ? blockIdx.x * 8 + warp : blockIdx.x; x < rows; x += few ? gridDim.x * 8 : gridDim.x) {
    const int tok = x / a.H, hd = x % a.H;
    const int64_t at = b * a.seq_parts + static_cast<int64_t>(hd / a.group) * all + tok * a.group + hd % a.group;
    float m = -INFINITY;
    for (int i = lane; i < c.splits; i += 32) m = fmaxf(m, a.part_ml[at + i * step].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float neg_m = m == -INFINITY ? 0.f : -m;
    __nv_bfloat16* dst = a.out + (q.row0 + tok) * a.out_pitch + static_cast<int64_t>(hd) * D;
    float l = 0.f;
    if (few) {
      float4 acc[V];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = 0; i < c.splits; ++i) {
        const float2 ml = a.part_ml[at + i * step];
        const float f = fast_exp2(ml.x + neg_m);
        l = fmaf(f, ml.y, l);
        const float4* src = reinterpret_cast<const float4*>(a.part_o + (at + i * step) * D);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float4 u = src[v * 32 + lane];
          acc[v].x = fmaf(f, u.x, acc[v].x), acc[v].y = fmaf(f, u.y, acc[v].y), acc[v].z = fmaf(f, u.z, acc[v].z), acc[v].w = fmaf(f, u.w, acc[v].w);
        }
      }
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
      for (int v = 0; v < V; ++v)
        *reinterpret_cast<uint2*>(dst + (v * 32 + lane) * 4) =
            make_uint2(pack_bf16x2(acc[v].x * inv, acc[v].y * inv), pack_bf16x2(acc[v].z * inv, acc[v].w * inv));
      if (a.lse && lane == 0) a.lse[static_cast<int64_t>(q.row0 + tok) * a.H + hd] = m + log2f(l);
    } else {
      const int grp = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = grp; i < c.splits; i += G) {
        const float2 ml = a.part_ml[at + i * step];
        const float f = fast_exp2(ml.x + neg_m);
        l = fmaf(f, ml.y, l);
        const float4 u = reinterpret_cast<const float4*>(a.part_o + (at + i * step) * D)[d];
        acc.x = fmaf(f, u.x, acc.x), acc.y = fmaf(f, u.y, acc.y), acc.z = fmaf(f, u.z, acc.z), acc.w = fmaf(f, u.w, acc.w);
      }
      part[grp][d] = acc;
      if (d == 0) part_l[grp] = l;
      __syncthreads();
      if (grp == 0) {
        l = part_l[0];
#pragma unroll
        for (int y = 1; y < G; ++y) {
          const float4 u = part[y][d];
          acc.x += u.x, acc.y += u.y, acc.z += u.z, acc.w += u.w;
          l += part_l[y];
        }
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        *reinterpret_cast<uint2*>(dst + d * 4) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        if (a.lse && d == 0) a.lse[static_cast<int64_t>(q.row0 + tok) * a.H + hd] = m + log2f(l);
      }
      __syncthreads();
    }
  }
}

// weights_out[b][g][j] = decay weights[b][g][j] + sum over the sequence's rows of kv head g of p(row, j), for j < len; a thread owns
// four keys, 256 apart, and adds their rows in order. Bound by reading the scores back (L2): 16 steps over up to 4 096 tokens (16 / 8 heads of
// 256) 80 us with the attention, 6 us of them here. Scores are written and read once because the attention cannot weigh a key before
// its row's last key is known; for a chunk they would be the larger part, so there they are computed again (paged_chunk.cu).
__global__ void __launch_bounds__(256) paged_weight_kernel(const PagedSeqs s, const PagedAttnArgs a, const PagedWeightArgs w, int* __restrict__ status) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, g = blockIdx.y;
  const PagedSeq q = paged_seq(s, b, status);
  const int first = blockIdx.x * 1024;
  if (first >= q.len || chunk_class(q, a)) return;
  const int all = q.nq * a.group, base = q.len - q.nq;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r = 0; r < all; ++r) {
    const int tok = r / a.group, hd = g * a.group + r % a.group, hi = base + tok, lo = a.window > 0 ? hi - a.window + 1 : 0;
    const float l = a.lse[static_cast<int64_t>(q.row0 + tok) * a.H + hd];
    const float lse = l == -INFINITY ? INFINITY : l;  // the row sees nothing, or all its scores are -inf: its output is 0, and it weighs nothing
    const float* src = a.scores + ((static_cast<int64_t>(b) * a.tok_cap + tok) * a.H + hd) * a.score_pitch + first + threadIdx.x;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int j = first + threadIdx.x + x * 256;
      if (j <= hi && j >= lo) sum[x] += fast_exp2(src[x * 256] - lse);
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int j = first + threadIdx.x + x * 256;
    if (j < q.len) {
      const float old = w.decay != 0.f ? w.in[b * w.in_seq + g * w.in_head + j] * w.decay : 0.f;
      w.out[b * w.out_seq + g * w.out_head + j] = old + sum[x];
    }
  }
}

// Finds the groups: runs of neighbouring sequences, none of them a long chunk, whose tables begin with the same pages. share[b]: key tiles of
// b's group (0: none), share[B + b]: behind a group's first sequence its end. One CTA: a warp compares two tables, then one thread walks
// the runs. A run ends where the common front changes by more than a factor of two (another content behind a prompt that both share),
// and a group whose units the workspace has no room for is left as it is.
__global__ void __launch_bounds__(1024) paged_share_kernel(const PagedSeqs s, const PagedAttnArgs a, int32_t* __restrict__ share, int units,
                                                           int* __restrict__ status) {
  __shared__ int lim[PG_MAX_SEQS], link[PG_MAX_SEQS], out[2 * PG_MAX_SEQS];
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int b = tid; b < s.B; b += 1024) {
    const PagedSeq q = paged_seq(s, b, status);
    lim[b] = q.nq > 0 && q.nq * a.group <= SHARE_ROWS * a.chunk_rows && q.len > q.nq ? (q.len - q.nq) / PG_TILE : 0;
    link[b] = out[b] = out[s.B + b] = 0;
  }
  __syncthreads();
  for (int b = warp; b + 1 < s.B; b += 32) {
    const int most = lim[b] < lim[b + 1] ? lim[b] : lim[b + 1];
    if (most < SHARE_TILES) continue;
    const int pages = (most * PG_TILE + (1 << s.page_log2) - 1) >> s.page_log2;
    const int32_t* x = s.table + b * s.table_pitch;
    const int32_t* y = x + s.table_pitch;
    int common = pages;
    for (int p0 = 0; p0 < pages && common == pages; p0 += 128) {
      bool same[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) same[u] = p0 + u * 32 + lane >= pages || x[p0 + u * 32 + lane] == y[p0 + u * 32 + lane];
#pragma unroll
      for (int u = 3; u >= 0; --u) {
        const uint32_t off = __ballot_sync(0xffffffffu, !same[u]);
        if (off) common = p0 + u * 32 + __ffs(off) - 1;
      }
    }
    const int64_t tiles = (static_cast<int64_t>(common) << s.page_log2) / PG_TILE;
    if (lane == 0) link[b] = tiles < most ? static_cast<int>(tiles) : most;
  }
  __syncthreads();
  if (tid == 0) {
    int used = 0, groups = 0;
    for (int b = 0; b + 1 < s.B;) {
      int t = link[b], e = b + 1;
      if (t < SHARE_TILES) {
        ++b;
        continue;
      }
      for (; e + 1 < s.B && link[e] >= SHARE_TILES && 2 * link[e] >= t && link[e] <= 2 * t; ++e) t = link[e] < t ? link[e] : t;
      if (!share_pays(e + 1 - b, t * PG_TILE, a.h, a.D)) {
        b = e;
        continue;
      }
      PagedSeq q;
      q.row0 = s.cu[b];
      q.nq = s.cu[e + 1] - q.row0;
      q.skip = t;
      q.cap = t * PG_TILE;
      q.len = q.cap + q.nq;
      const int need = chunk_cut(q, a).units;
      if (used + need <= units) {
        used += need;
        ++groups;
        for (int i = b; i <= e; ++i) out[i] = t;
        out[s.B + b] = e + 1;
      }
      b = e + 1;
    }
    share[2 * s.B] = groups;
  }
  __syncthreads();
  for (int i = tid; i < 2 * s.B; i += 1024) share[i] = out[i];
}

// A sequence with more rows per kv head than this is the chunk kernels', where a head set of it fills 256-row items: measured on 32
// sequences of 2 000 tokens (16 / 8 heads of 256) 32 rows took 138 us in the few-row kernel and 168 there, 64 rows 253 and 172; with
// three head sets per kv head (24 / 4 heads) 48 rows 106 and 237, 96 rows 250 and 240.
// Where the slots' weights are kept the border is 32 rows for any number of head sets: the few-row kernel's scores go out to memory and back,
// the chunk kernels' second product costs less (24 / 4 heads of 256: three sequences of 14 tokens over 275 67 us there, 38 here; five of up to
// 23 over up to 3 656, window 1 024, 132 and 85).
__host__ __device__ constexpr int chunk_rows_of(int group, bool weights) { return weights ? 32 : 32 * (group >> chunk_heads_log2(group)); }

// what a call needs: sizes of the workspace's parts in bytes (256-byte multiples)
struct PagedSizes {
  int64_t seq_parts, part_o, part_ml, chunk_o, chunk_ml, joins, share, lse, scores, total;
  int64_t score_pitch;
  int tok_cap, chunk_rows, max_units, share_units, unit_slots;
  bool too_large;
};
static int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
// alone: the call has one sequence (B: those of a launch); window 0: none
static PagedSizes paged_sizes(int64_t n, int64_t B, int H, int h, int D, int64_t max_q, int64_t max_len, int64_t window, bool weights, bool shared, bool alone) {
  PagedSizes z = {};
  // key tiles that so many neighbouring rows see at most: their window's slots, wherever in a tile they begin
  const auto seen = [=](int64_t rows, int64_t tiles) {
    const int64_t w = window > 0 ? (rows - 1 + window + 2 * PG_TILE - 2) / PG_TILE : tiles;
    return w < tiles ? w : tiles;
  };
  const int64_t tiles = (max_len + PG_TILE - 1) / PG_TILE;
  const int64_t group = H / h;
  z.chunk_rows = chunk_rows_of(static_cast<int>(group), weights);
  const int64_t most = z.chunk_rows / group;  // tokens of a sequence that is not the chunk kernel's
  const int64_t few = seen(max_q < most ? max_q : most, tiles);
  const int64_t slots = few < PG_SMS / h ? few : PG_SMS / h;  // most splits of a sequence
  const bool chunk_only = alone && max_q > most;  // the few-row kernels are not launched
  if (slots > 1 && !chunk_only) {
    const int64_t by_rows = (max_q < most ? max_q : most) * H * slots;  // every row in every split
    const int64_t by_items = static_cast<int64_t>(PG_SMS) * RT;  // every free slot one full row tile
    z.seq_parts = by_rows < by_items ? by_rows : by_items;
  }
  shared = shared && !weights && B > 1 && tiles > SHARE_TILES && share_pays(B, max_len, h, D);
  if (shared) {  // a sequence of a group leaves parts in any case
    const int64_t one = (max_q < SHARE_ROWS * most ? max_q : SHARE_ROWS * most) * H;
    const int64_t parts = one * (slots < 1 ? 1 : slots < PG_SKIP_SPLITS ? slots : PG_SKIP_SPLITS);
    z.seq_parts = z.seq_parts > parts ? z.seq_parts : parts;
  }
  z.part_o = up256(B * z.seq_parts * D * 4);
  z.part_ml = up256(B * z.seq_parts * 8);
  const int hl = chunk_heads_log2(static_cast<int>(group)), tl = 8 - hl;
  const int64_t most_units = chunk_units_of(D), per_tt = H >> hl, ntt = (max_q + (1 << tl) - 1) >> tl;
  // items of one token tile (and fronts) are cut into parts, a unit each: one slot of 256 rows; other units end one item and begin the next
  z.unit_slots = ntt <= 1 && per_tt <= most_units ? 1 : 2;
  int64_t all_units = 0;
  if (max_q > most) {
    const int64_t each = seen(max_q < 1 << tl ? max_q : 1 << tl, tiles), work = ntt * per_tt * (each > 0 ? each : 1);
    if (work >= (1ll << 31)) z.too_large = true;  // the chunk kernels count (item, key tile) pairs in 32 bits
    // (an item makes a unit, or a unit holds CHUNK_MIN_TILES pairs, or a part of an item four)
    int64_t units = work / 4 + ntt * per_tt;
    if (z.unit_slots == 1) {
      const int64_t parts = most_units / per_tt < each / 4 ? most_units / per_tt : each / 4;
      units = per_tt * (parts > 1 ? parts : 1);
    }
    units = units > most_units ? most_units : units;
    const int64_t seqs = B == 1 ? 1 : n / (most + 1) < B ? n / (most + 1) : B;  // so many can be the chunk kernel's
    all_units = seqs * units;
  }
  if (shared) {
    // a unit per item of a group, or up to one per CTA (pair) for a group of few items: room for four such groups
    const int64_t items = ((n >> tl) + B / 2) * per_tt + 4 * most_units;
    z.share_units = static_cast<int>(items < 4 * PG_SMS ? items : 4 * PG_SMS);
    z.share = up256(B * 8 + 4);
    all_units += z.share_units;
  }
  z.max_units = static_cast<int>(all_units);
  if (all_units > 0) {
    z.chunk_o = up256(all_units * z.unit_slots * 256 * D * 4);
    z.chunk_ml = up256(all_units * z.unit_slots * 256 * 8);
    z.joins = up256(all_units * static_cast<int64_t>(sizeof(ChunkJoin)) + 16);
  }
  if (weights) z.lse = up256(n * H * 4);
  if (weights && !chunk_only) {
    z.score_pitch = tiles * PG_TILE;
    z.tok_cap = static_cast<int>(max_q < most ? max_q : most);
    z.scores = up256(B * z.tok_cap * H * z.score_pitch * 4);
  }
  z.total = z.part_o + z.part_ml + z.chunk_o + z.chunk_ml + z.joins + z.share + z.lse + z.scores;
  return z;
}

// Parts are sized for every sequence of a launch at once (1 024 of 40 new tokens over 4 096 would ask for 21 GB), so a call of many
// sequences is made in launches of as many as this holds, one behind the other over the same workspace: by then each of them fills the GPU many
// times over. A sequence's cuts are its own, so its results stay the same; a common front ends where a launch ends.
static constexpr int64_t PG_ROOM = 2ll << 30;
struct PagedPlan {
  PagedSizes z;
  int64_t seqs;  // of a launch
};
static PagedPlan paged_plan(int64_t n, int64_t B, int H, int h, int D, int64_t max_q, int64_t max_len, int64_t window, bool weights, bool shared, int64_t room) {
  PagedPlan p = {paged_sizes(n, B, H, h, D, max_q, max_len, window, weights, shared, B == 1), B};
  int64_t launches = 1;
  while (p.seqs > 1 && p.z.total - p.z.lse > room) {
    const int64_t by_size = (p.z.total - p.z.lse) * launches / room;  // (rounded down: the least that could do)
    launches = by_size > launches ? by_size : launches + 1;
    p.seqs = (B + launches - 1) / launches;
    p.z = paged_sizes(n, p.seqs, H, h, D, max_q, max_len, window, weights, shared, false);
  }
  return p;
}
// what the caller has been told to bring knows no window
static PagedPlan paged_plan(int64_t n, int64_t B, int H, int h, int D, int64_t max_q, int64_t max_len, bool weights, bool shared) {
  return paged_plan(n, B, H, h, D, max_q, max_len, 0, weights, shared, PG_ROOM);
}

template <int D>
static int launch_paged(const PagedPool& kp, const PagedPool& vp, const PagedSeqs& s, const PagedAttnArgs& a, const PagedWeightArgs* w, int64_t max_q,
                        int max_splits, int share_units, cudaStream_t st, int dev, int* status) {
  CUtensorMap tmK, tmV;
  int r;
  const uint32_t box = kp.page < 64 ? static_cast<uint32_t>(kp.page) : 64u;
  if ((r = make_tmap_pages(&tmK, kp, box, D / 64)) || (r = make_tmap_pages(&tmV, vp, box, D / 64))) return r;
  static std::atomic<bool> attr_set[64];
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    SPINF_CUDA_OK(cudaFuncSetAttribute(paged_step_kernel<D, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, StepSmem<D>::TOTAL));
    SPINF_CUDA_OK(cudaFuncSetAttribute(paged_step_kernel<D, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, StepSmem<D>::TOTAL));
    SPINF_CUDA_OK(cudaFuncSetAttribute(paged_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsSmem<D>::TOTAL));
    attr_set[dev].store(true, std::memory_order_release);
  }
  const unsigned grid = static_cast<unsigned>(sm_count());
  // with one sequence its kernel is known here: the others' launches fall away
  const bool step = a.only ? a.only == 1 : true, rows = a.only ? a.only == 2 : max_q * a.group > STEP_ROWS;
  const bool chunk = a.only ? a.only == 3 : max_q * a.group > a.chunk_rows || share_units > 0;
  if (share_units > 0) {
    PagedSeqs plain = s;
    plain.share = nullptr;
    ++paged_launches;
    paged_share_kernel<<<1, 1024, 0, st>>>(plain, a, const_cast<int32_t*>(s.share), share_units, status);
    SPINF_CUDA_OK(cudaGetLastError());
  }
  if (step) {
    const auto kern = max_q * a.group <= 8 ? paged_step_kernel<D, 1> : paged_step_kernel<D, 2>;
    SPINF_CUDA_OK(launch_after(kern, dim3(grid), dim3(step_threads(D)), st, StepSmem<D>::TOTAL, 1, share_units > 0, tmK, tmV, s, a, status));
  }
  if (rows) SPINF_CUDA_OK(launch_after(paged_rows_kernel<D>, dim3(grid), dim3(ROWS_THREADS), st, RowsSmem<D>::TOTAL, 1, step, tmK, tmV, s, a, status));
  if (max_splits > 1 && (step || rows)) {
    const int64_t most = a.chunk_rows / a.group;  // tokens of a sequence that is not the chunk kernel's
    int64_t gx = (max_q < most ? max_q : most) * a.H;
    const int64_t fill = 8 * PG_SMS / s.B > 16 ? 8 * PG_SMS / s.B : 16;  // (CTAs of many sequences that have nothing to join cost 10 us to start)
    if (gx > fill) gx = fill;
    SPINF_CUDA_OK(launch_after(paged_join_kernel<D>, dim3(static_cast<unsigned>(gx), s.B), dim3(256), st, 0, 1, true, s, a, status));
  }
  if (chunk && (r = paged_chunk_launch(D, kp, vp, s, a, w, step || rows, st, dev, status))) return r;
  if (w && a.only != 3 && s.max_len > 0)
    SPINF_CUDA_OK(launch_after(paged_weight_kernel, dim3(static_cast<unsigned>((s.max_len + 1023) / 1024), a.h, s.B), dim3(256), st, 0, 1, true, s, a, *w, status));
  return 0;
}

}  // namespace spinf

using namespace spinf;

extern "C" int64_t spinf_paged_attention_workspace_bytes(int64_t n, int64_t B, int32_t H, int32_t Hkv, int32_t D, int64_t max_q, int64_t max_len,
                                                         int32_t weights, int32_t shared) {
  if (B > PG_MAX_SEQS) return SPINF_ERR_TOO_LARGE;
  if (n < 0 || B < 0 || H <= 0 || Hkv <= 0 || H % Hkv || (D != 128 && D != 256) || max_q < 0 || max_len < 0) return SPINF_ERR_BAD_ARGUMENT;
  const PagedSizes z = paged_plan(n, B, H, Hkv, D, max_q < n ? max_q : n, max_len, weights != 0, shared != 0).z;
  return z.too_large ? SPINF_ERR_TOO_LARGE : z.total;
}

extern "C" int spinf_paged_attention(const void* q, int64_t q_pitch, int64_t n, int32_t H, int32_t Hkv, int32_t D, const void* k_pages,
                                     const void* v_pages, int64_t n_pages, int32_t page, const int64_t* k_strides_host,
                                     const int64_t* v_strides_host, const int32_t* table, int64_t table_pitch, const int32_t* lens,
                                     const int32_t* cu, int32_t B, int64_t max_q, int64_t max_len, int32_t window, int32_t shared, float scale,
                                     const float* weights_in, float* weights_out, const int64_t* weight_strides_host, float decay,
                                     void* out, int64_t out_pitch, void* workspace, int64_t workspace_bytes, void* stream) {
  paged_launches = 0;
  if (B == 0 || (n == 0 && !weights_out)) return 0;  // nothing to do: the row pointers may be null
  SPINF_CHECK_ARG(k_pages && v_pages && k_strides_host && v_strides_host && table && lens && cu && n >= 0 && B > 0);
  SPINF_CHECK_ARG(n == 0 || (q && out));
  SPINF_CHECK_ARG(H > 0 && Hkv > 0 && H % Hkv == 0 && H <= 1024 && (D == 128 || D == 256) && n < (1ll << 31) / H);
  SPINF_CHECK_ARG(q_pitch >= static_cast<int64_t>(H) * D && out_pitch >= static_cast<int64_t>(H) * D && q_pitch % 8 == 0 && out_pitch % 8 == 0);
  SPINF_CHECK_ARG(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0);
  SPINF_CHECK_ARG(page >= 16 && page <= 256 && (page & (page - 1)) == 0 && n_pages > 0 && n_pages < (1ll << 31));
  SPINF_CHECK_ARG(max_q >= 0 && max_len >= 0 && max_len <= table_pitch * page && max_len < (1ll << 30) && window >= 0 && scale > 0.f);
  SPINF_CHECK_ARG(!weights_out || (weight_strides_host && (weights_in || decay == 0.f)));
  if (B > PG_MAX_SEQS) return SPINF_ERR_TOO_LARGE;
  const int64_t mq = max_q < n ? max_q : n;
  const bool narrow = window > 0 && window < max_len;  // (a window of max_len slots holds everything: no window)
  PagedPlan plan = paged_plan(n, B, H, Hkv, D, mq, max_len, weights_out != nullptr, shared != 0);
  if (narrow) plan = paged_plan(n, B, H, Hkv, D, mq, max_len, window, weights_out != nullptr, false, plan.z.total - plan.z.lse);  // more sequences fit in
  const PagedSizes& z = plan.z;
  if (z.too_large) return SPINF_ERR_TOO_LARGE;
  SPINF_CHECK_ARG(z.total == 0 || (workspace && workspace_bytes >= z.total && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0));
  int dev = 0;
  SPINF_CUDA_OK(cudaGetDevice(&dev));
  int* status = status_word(dev);
  if (!status) return SPINF_ERR_CUDA;
  PagedSeqs s = {};
  s.table = table;
  s.table_pitch = table_pitch;
  s.lens = lens;
  s.cu = cu;
  s.n_pages = static_cast<int>(n_pages);
  s.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  s.max_len = static_cast<int>(max_len);
  s.max_q = static_cast<int>(mq);
  s.n = n;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PagedAttnArgs a = {};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_pitch = q_pitch;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.out_pitch = out_pitch;
  a.H = H;
  a.h = Hkv;
  a.D = D;
  a.group = H / Hkv;
  a.window = narrow ? window : 0;  // (sums with it stay in 32 bits)
  a.hp_log2 = chunk_heads_log2(a.group);
  a.sets = a.group >> a.hp_log2;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.seq_parts = z.seq_parts;
  a.chunk_rows = z.chunk_rows;
  a.only = B == 1 && mq > 0 ? class_of(mq * a.group, z.chunk_rows) : 0;
  a.unit_slots = z.unit_slots;
  a.max_units = z.max_units;
  a.fronts_only = z.share_units > 0 && mq * a.group <= z.chunk_rows;
  auto take = [&](int64_t bytes) {
    uint8_t* p = ws;
    ws += bytes;
    return p;
  };
  a.part_o = reinterpret_cast<float*>(take(z.part_o));
  a.part_ml = reinterpret_cast<float2*>(take(z.part_ml));
  a.chunk_o = reinterpret_cast<float*>(take(z.chunk_o));
  a.chunk_ml = reinterpret_cast<float2*>(take(z.chunk_ml));
  a.n_units = reinterpret_cast<int32_t*>(take(z.joins));
  a.joins = reinterpret_cast<ChunkJoin*>(a.n_units + 4);
  if (z.share_units) s.share = reinterpret_cast<int32_t*>(take(z.share));
  if (weights_out) {
    a.lse = reinterpret_cast<float*>(take(z.lse));
    a.scores = reinterpret_cast<float*>(take(z.scores));
    a.score_pitch = z.score_pitch;
    a.tok_cap = z.tok_cap;
  }
  PagedWeightArgs w;
  if (weights_out) {
    w.in = weights_in;
    w.out = weights_out;
    w.in_seq = weight_strides_host[0], w.in_head = weight_strides_host[1];
    w.out_seq = weight_strides_host[2], w.out_head = weight_strides_host[3];
    w.decay = decay;
  }
  const PagedPool kp = {k_pages, n_pages, page, Hkv, D, k_strides_host[0], k_strides_host[1], k_strides_host[2]};
  const PagedPool vp = {v_pages, n_pages, page, Hkv, D, v_strides_host[0], v_strides_host[1], v_strides_host[2]};
  const int max_splits = z.seq_parts ? 2 : 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int64_t b = 0; b < B; b += plan.seqs) {
    s.B = static_cast<int>(plan.seqs < B - b ? plan.seqs : B - b);
    s.table = table + b * table_pitch;
    s.lens = lens + b;
    s.cu = cu + b;
    if (weights_out) {
      w.in = weights_in ? weights_in + b * w.in_seq : nullptr;
      w.out = weights_out + b * w.out_seq;
    }
    const int r = D == 256 ? launch_paged<256>(kp, vp, s, a, weights_out ? &w : nullptr, mq, max_splits, z.share_units, st, dev, status)
                           : launch_paged<128>(kp, vp, s, a, weights_out ? &w : nullptr, mq, max_splits, z.share_units, st, dev, status);
    if (r) return r;
  }
  return 0;
}

extern "C" int64_t spinf_paged_launches(void) { return paged_launches; }
