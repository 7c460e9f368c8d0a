// What the kernels over the paged K/V cache share: the call's sequences as they lie in device memory, the rule that cuts a
// sequence's keys into splits, and the list of work items every CTA builds for itself.
//
// A sequence of a call has nq new rows (rows cu[b] .. cu[b + 1] of q) and `len` cached tokens, the new ones included; row i sits in
// cache slot len - nq + i and sees the slots up to its own, with a window only the last `window` of them. Slot s lies in page
// table[b][s / page], row s % page. A pool of pages is [pages, kv heads, page, D] with any strides between pages, heads and rows.
#pragma once
#include "common.cuh"
#include "host_util.h"
#include "paged_pool.h"

namespace spinf {

static constexpr int PG_TILE = 128;      // keys per tile
static constexpr int PG_MAX_SEQS = 1024;  // sequences of a call: their item counts are scanned in shared memory
static constexpr int PG_SMS = 148;       // what the split rule fills (a constant, not the device's count: results depend on it)

struct PagedSeqs {
  const int32_t* table;
  int64_t table_pitch;
  const int32_t* lens;
  const int32_t* cu;
  int B, n_pages, page_log2;
  int max_len;  // longest sequence the caller's buffers are sized for
  int max_q;    // most new rows of a sequence they are sized for
  int64_t n;    // rows of q
  const int32_t* share;  // [2][B] and the number of groups, or null: key tiles of each sequence that its group reads together; behind a group's first, at B + b, its end
};

struct PagedSeq {
  int row0, nq, len;
  int skip;  // key tiles at the front that are another item's work (0: none)
  int cap;   // slots from here on are another item's work (a group's common front; INT_MAX otherwise)
};
static constexpr int PG_NO_CAP = 0x7fffffff;
static constexpr int PG_SKIP_SPLITS = 4;  // most splits behind a shared front: little is left there, and the parts of up to four times the rows take room

// the sequence's numbers, cut to what the buffers hold: one that lies outside them is reported and treated as
// shorter, or as having no new rows
__device__ __forceinline__ PagedSeq paged_seq(const PagedSeqs& s, int b, int* status) {
  PagedSeq r;
  const int r0 = s.cu[b], r1 = s.cu[b + 1];
  r.len = s.lens[b];
  r.row0 = r0;
  r.nq = r1 - r0;
  r.skip = s.share ? s.share[b] : 0;
  r.cap = PG_NO_CAP;
  if (r0 < 0 || r1 < r0 || r1 > s.n || r.nq > s.max_q) {
    r.row0 = r.nq = 0;
    atomicCAS(status, 0, ST_BAD_INDEX);
  }
  if (r.len < 0 || r.len > s.max_len) {
    r.len = r.len < 0 ? 0 : s.max_len;
    atomicCAS(status, 0, ST_BAD_INDEX);
  }
  return r;
}

// How a sequence's work is cut. Everything here follows from the sequence's own lengths and the model's heads, so a sequence's
// result does not depend on what else is in the call.
struct PagedCut {
  int row_tiles;  // tiles of `tile_rows` query rows of one key / value head
  int t_lo, t_hi;  // key tiles any row sees
  int splits, tiles_per_split;
};

// items_per_split: work items one split of the sequence makes (kv heads x row tiles); slots: items the GPU runs at once. One split
// per free slot: more would only add partial results to join, fewer leave SMs idle.
__device__ __forceinline__ PagedCut paged_cut(const PagedSeq& q, int window, int row_tiles, int items_per_split, int slots, int min_tiles) {
  PagedCut c;
  c.row_tiles = row_tiles;
  const int first = q.len - q.nq + 1 - window;
  c.t_lo = window > 0 && first > 0 ? first / PG_TILE : q.skip;
  c.t_hi = (q.len + PG_TILE - 1) / PG_TILE;
  const int tiles = c.t_hi > c.t_lo ? c.t_hi - c.t_lo : 0;
  int s = slots / (items_per_split > 0 ? items_per_split : 1);
  s = s < tiles / min_tiles ? s : tiles / min_tiles;
  s = s < 1 ? 1 : q.skip && s > PG_SKIP_SPLITS ? PG_SKIP_SPLITS : s;
  c.tiles_per_split = (tiles + s - 1) / s;
  c.splits = c.tiles_per_split > 0 ? (tiles + c.tiles_per_split - 1) / c.tiles_per_split : 1;
  return c;
}

// exclusive prefix sums of `count(b)` over the sequences into pre[0 .. B] (shared memory); every thread of the CTA takes part
template <class Count>
__device__ __forceinline__ void paged_item_prefix(int B, int* pre, int nthreads, Count count) {
  for (int b = threadIdx.x; b < B; b += nthreads) pre[b + 1] = count(b);
  if (threadIdx.x == 0) pre[0] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    int carry = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
      const int b = b0 + static_cast<int>(threadIdx.x);
      int v = b < B ? pre[b + 1] : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (static_cast<int>(threadIdx.x) >= o) v += u;
      }
      if (b < B) pre[b + 1] = v + carry;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
}

// the sequence item `it` belongs to: the largest b with pre[b] <= it (it < pre[B])
__device__ __forceinline__ int paged_find(const int* pre, int B, int it) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= it) lo = mid;
    else hi = mid;
  }
  return lo;
}

// programmatic dependent launch: the next kernel of the chain may start its CTAs (they wait in pdl_wait until this one is done)
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, int c4, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

// a launch that, with `early`, may start before the kernel ahead of it on the stream has ended (its pdl_wait holds it back); the first
// kernel of a call must not: what is ahead of it is not ours
template <class... Params, class... Args>
inline cudaError_t launch_after(void (*kern)(Params...), dim3 grid, dim3 block, cudaStream_t st, int smem, int cluster, bool early, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = early ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  ++paged_launches;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace spinf
