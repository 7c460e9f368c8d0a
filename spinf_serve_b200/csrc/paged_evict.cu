// Eviction from the paged K/V cache by accumulated attention weight: per sequence and key / value head the last `recent` slots stay,
// of the others the keep - recent with the largest weight (ties: the lowest slot first; a NaN counts as less than every number); what
// stays moves, in slot order, to the pages of new_table.
//
//   paged_select_kernel  one CTA per (sequence, kv head): radix select over the weights' bits as ordered integers (11, 11 and 10 bits,
//                        a histogram in shared memory each), then the slots above the threshold, and the first of those equal to it,
//                        in ascending order: every warp counts and then writes one contiguous segment
//   paged_move_kernel    the kept rows of K and V, 16 bytes a lane, several rows of a warp in flight: the bytes that bound the call.
//                        16 sequences of up to 16 000 tokens to 4 096 (16 kv heads of 128): 214 us, 1.1 GB at 5.1 TB/s; 4 of 2 049
//                        to 1 024 (8 of 256): 15.5 us, the select's chain of three passes and the move behind it
#include "paged.cuh"

namespace spinf {

struct EvictArgs {
  const float* weights;  // [B][h][..], or null: only `recent` decides
  int64_t w_seq, w_head;
  int keep, recent, h;
  int32_t* kept;      // [B][h][keep], -1 behind the last
  float* w_out;       // [B][h][keep], 0 behind the last (null without weights)
  int32_t* new_lens;  // [B]
  const int32_t* new_table;
  int64_t new_pitch;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;
};

static constexpr int SEL_THREADS = 1024;

__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 counts as +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(SEL_THREADS) paged_select_kernel(const PagedSeqs s, const EvictArgs a, int* __restrict__ status) {
  __shared__ int hist[2048];
  __shared__ int warp_sum[32];
  __shared__ int found[2];  // bin, candidates above it
  __shared__ int seg_gt[33], seg_eq[33];
  pdl_trigger();
  const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int len = s.lens[b];
  if (len < 0 || len > s.max_len) {
    len = len < 0 ? 0 : s.max_len;
    if (tid == 0) atomicCAS(status, 0, ST_BAD_INDEX);
  }
  const float* w = a.weights ? a.weights + b * a.w_seq + g * a.w_head : nullptr;
  const int64_t out0 = (static_cast<int64_t>(b) * a.h + g) * a.keep;
  int32_t* kept = a.kept + out0;
  float* w_out = a.w_out ? a.w_out + out0 : nullptr;
  if (g == 0 && tid == 0) a.new_lens[b] = len < a.keep ? len : a.keep;
  if (len <= a.keep) {
    for (int i = tid; i < a.keep; i += SEL_THREADS) {
      kept[i] = i < len ? i : -1;
      if (w_out) w_out[i] = i < len ? w[i] : 0.f;
    }
    return;
  }
  const int m = len - a.recent, quota = a.keep - a.recent;  // candidates [0, m), m > quota
  for (int i = tid; i < a.recent; i += SEL_THREADS) {
    kept[quota + i] = m + i;
    if (w_out) w_out[quota + i] = w[m + i];
  }
  if (quota == 0) return;
  // the quota-th largest key, 11 + 11 + 10 bits
  uint32_t prefix = 0;
  int need = quota;  // candidates still to be found among those that share the prefix
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < 2048; i += SEL_THREADS) hist[i] = 0;
    __syncthreads();
    const uint32_t mask = (1u << bits) - 1u;
    for (int i0 = tid; i0 < m; i0 += 4 * SEL_THREADS) {
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = i0 + u * SEL_THREADS < m ? w[i0 + u * SEL_THREADS] : 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t key = order_key(x[u]);
        if (i0 + u * SEL_THREADS < m && (pass == 0 || (key >> (shift + bits)) == prefix)) atomicAdd(&hist[(key >> shift) & mask], 1);
      }
    }
    __syncthreads();
    // counts from the top: thread t holds bins 2047 - 2 t and 2046 - 2 t
    const int c0 = hist[2047 - 2 * tid], c1 = hist[2046 - 2 * tid];
    int incl = c0 + c1;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      int v = warp_sum[lane];
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      warp_sum[lane] = v;
    }
    __syncthreads();
    const int above = incl - c0 - c1 + (warp ? warp_sum[warp - 1] : 0);
    if (above < need && above + c0 >= need) found[0] = 2047 - 2 * tid, found[1] = above;
    else if (above + c0 < need && above + c0 + c1 >= need) found[0] = 2046 - 2 * tid, found[1] = above + c0;
    __syncthreads();
    prefix = (prefix << bits) | static_cast<uint32_t>(found[0]);
    need -= found[1];
    __syncthreads();
  }
  // keys above `prefix` stay, and the first `need` of those equal to it
  const int seg = ((m + 31) / 32 + 31) / 32 * 32;
  const int i_lo = warp * seg, i_hi = i_lo + seg < m ? i_lo + seg : m;
  int gt = 0, eq = 0;
  for (int i0 = i_lo; i0 < i_hi; i0 += 128) {
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = i0 + u * 32 + lane < i_hi ? w[i0 + u * 32 + lane] : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in = i0 + u * 32 + lane < i_hi;
      const uint32_t key = order_key(x[u]);
      gt += in && key > prefix;
      eq += in && key == prefix;
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  if (lane == 0) seg_gt[warp + 1] = gt, seg_eq[warp + 1] = eq;
  if (tid == 0) seg_gt[0] = seg_eq[0] = 0;
  __syncthreads();
  if (tid == 0)
    for (int i = 1; i <= 32; ++i) seg_gt[i] += seg_gt[i - 1], seg_eq[i] += seg_eq[i - 1];
  __syncthreads();
  int n_gt = seg_gt[warp], n_eq = seg_eq[warp];
  const uint32_t below = (1u << lane) - 1u;
  for (int i0 = i_lo; i0 < i_hi; i0 += 128) {
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = i0 + u * 32 + lane < i_hi ? w[i0 + u * 32 + lane] : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * 32 + lane;
      const bool in = i < i_hi;
      const uint32_t key = order_key(x[u]);
      const uint32_t bg = __ballot_sync(0xffffffffu, in && key > prefix), be = __ballot_sync(0xffffffffu, in && key == prefix);
      const int my_eq = n_eq + __popc(be & below);
      const bool stay = in && (key > prefix || (key == prefix && my_eq < need));
      if (stay) {
        const int at = n_gt + __popc(bg & below) + (my_eq < need ? my_eq : need);
        kept[at] = i;
        if (w_out) w_out[at] = x[u];
      }
      n_gt += __popc(bg);
      n_eq += __popc(be);
    }
  }
}

// Row blocks from the last one down, all sequences and heads of a block before the next: the `recent` rows, and all rows of a sequence
// that keeps everything, move while the select is still at work; only the others wait for its answer.
template <int D>
__global__ void __launch_bounds__(256) paged_move_kernel(const PagedSeqs s, const EvictArgs a, int blocks, int* __restrict__ status) {
  constexpr int LANES = D / 8, GROUPS = 256 / LANES, IPT = 4;
  const int per_block = s.B * a.h;
  const int blk = blocks - 1 - static_cast<int>(blockIdx.x / per_block), bg = static_cast<int>(blockIdx.x % per_block);
  const int b = bg / a.h, g = bg - b * a.h, sub = threadIdx.x % LANES, group = threadIdx.x / LANES;
  int len = s.lens[b];
  len = len < 0 ? 0 : len > s.max_len ? s.max_len : len;  // (reported by the select)
  const int quota = len > a.keep ? a.keep - a.recent : 0;  // rows the select chooses
  const int shift = len > a.keep ? len - a.keep : 0;       // the others: old slot = row + shift
  const int first = blk * GROUPS * IPT, i0 = first + group * IPT;
  const bool wait = first < quota;
  if (wait) pdl_wait();
  const int32_t* kept = a.kept + (static_cast<int64_t>(b) * a.h + g) * a.keep;
  const int in_page = (1 << s.page_log2) - 1, rows = len < a.keep ? len : a.keep;
  uint4 k[IPT], v[IPT];
  int to[IPT];
#pragma unroll
  for (int x = 0; x < IPT; ++x) {
    const int slot = i0 + x >= rows ? -1 : i0 + x < quota ? kept[i0 + x] : i0 + x + shift;
    to[x] = -1;
    if (slot < 0) continue;
    const int src = s.table[b * s.table_pitch + (slot >> s.page_log2)], dst = a.new_table[b * a.new_pitch + ((i0 + x) >> s.page_log2)];
    if (src < 0 || src >= s.n_pages || dst < 0 || dst >= s.n_pages) {
      if (sub == 0) atomicCAS(status, 0, ST_BAD_INDEX);
      continue;
    }
    to[x] = dst;
    k[x] = *reinterpret_cast<const uint4*>(a.k + src * a.k_page + g * a.k_head + (slot & in_page) * a.k_row + sub * 8);
    v[x] = *reinterpret_cast<const uint4*>(a.v + src * a.v_page + g * a.v_head + (slot & in_page) * a.v_row + sub * 8);
  }
#pragma unroll
  for (int x = 0; x < IPT; ++x) {
    if (to[x] < 0) continue;
    const int64_t row = (i0 + x) & in_page;
    *reinterpret_cast<uint4*>(const_cast<__nv_bfloat16*>(a.k) + to[x] * a.k_page + g * a.k_head + row * a.k_row + sub * 8) = k[x];
    *reinterpret_cast<uint4*>(const_cast<__nv_bfloat16*>(a.v) + to[x] * a.v_page + g * a.v_head + row * a.v_row + sub * 8) = v[x];
  }
  if (!wait) pdl_wait();  // this kernel's end is the call's: not before the select's
}

}  // namespace spinf

using namespace spinf;

extern "C" int spinf_paged_evict(void* k_pages, void* v_pages, int64_t n_pages, int32_t page, int32_t Hkv, int32_t D,
                                 const int64_t* k_strides_host, const int64_t* v_strides_host, const int32_t* table, int64_t table_pitch,
                                 const int32_t* lens, int32_t B, int64_t max_len, const float* weights, int64_t w_seq, int64_t w_head,
                                 int64_t keep, int64_t recent, const int32_t* new_table, int64_t new_pitch, int32_t* new_lens,
                                 int32_t* kept, float* weights_out, void* stream) {
  paged_launches = 0;
  if (B == 0) return 0;  // nothing to do: the pointers may be null
  SPINF_CHECK_ARG(k_pages && v_pages && k_strides_host && v_strides_host && table && lens && new_table && new_lens && kept && B > 0);
  SPINF_CHECK_ARG(Hkv > 0 && (D == 128 || D == 256) && n_pages > 0 && n_pages < (1ll << 31));
  SPINF_CHECK_ARG(page >= 16 && page <= 256 && (page & (page - 1)) == 0);
  SPINF_CHECK_ARG(max_len >= 0 && max_len <= table_pitch * page && max_len < (1ll << 30));
  SPINF_CHECK_ARG(keep > 0 && recent >= 0 && recent <= keep && keep <= new_pitch * page && keep < (1ll << 30));
  SPINF_CHECK_ARG((weights != nullptr) == (weights_out != nullptr) && (weights || recent == keep));
  if (B > 65535 || Hkv > 65535 || (keep / (32 * 256 / D) + 1) * Hkv * B >= (1ll << 31)) return SPINF_ERR_TOO_LARGE;
  uintptr_t bits = reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages);
  for (int i = 0; i < 3; ++i) bits |= static_cast<uintptr_t>(k_strides_host[i] | v_strides_host[i]) * 2;
  SPINF_CHECK_ARG((bits & 15) == 0);  // rows move 16 bytes at a time
  int dev = 0;
  SPINF_CUDA_OK(cudaGetDevice(&dev));
  int* status = status_word(dev);
  if (!status) return SPINF_ERR_CUDA;
  PagedSeqs s = {};
  s.table = table;
  s.table_pitch = table_pitch;
  s.lens = lens;
  s.B = B;
  s.n_pages = static_cast<int>(n_pages);
  s.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  s.max_len = static_cast<int>(max_len);
  EvictArgs a;
  a.weights = weights;
  a.w_seq = w_seq, a.w_head = w_head;
  a.keep = static_cast<int>(keep), a.recent = static_cast<int>(recent), a.h = Hkv;
  a.kept = kept;
  a.w_out = weights_out;
  a.new_lens = new_lens;
  a.new_table = new_table;
  a.new_pitch = new_pitch;
  a.k = static_cast<const __nv_bfloat16*>(k_pages);
  a.v = static_cast<const __nv_bfloat16*>(v_pages);
  a.k_page = k_strides_host[0], a.k_head = k_strides_host[1], a.k_row = k_strides_host[2];
  a.v_page = v_strides_host[0], a.v_head = v_strides_host[1], a.v_row = v_strides_host[2];
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ++paged_launches;
  paged_select_kernel<<<dim3(Hkv, B), SEL_THREADS, 0, st>>>(s, a, status);
  SPINF_CUDA_OK(cudaGetLastError());
  const int64_t per_cta = (256 / (D / 8)) * 4, blocks = (keep + per_cta - 1) / per_cta;
  const dim3 grid(static_cast<unsigned>(blocks * Hkv * B));
  SPINF_CUDA_OK(D == 256 ? launch_after(paged_move_kernel<256>, grid, dim3(256), st, 0, 1, true, s, a, static_cast<int>(blocks), status)
                         : launch_after(paged_move_kernel<128>, grid, dim3(256), st, 0, 1, true, s, a, static_cast<int>(blocks), status));
  return 0;
}
