// Append of a step's rows to the paged K/V cache: per-head RMSNorm of q / k (with weight) and v (without), rotary embedding of q / k,
// q to a dense output, k and v straight to their cache slots, in one pass over the fused projection's rows.
//   r = rsqrt(mean(x^2) + eps),  y = x r w,  y1' = y1 cos - y2 sin,  y2' = y2 cos + y1 sin  (halves of the rotary dimensions)
// Everything in fp32 with one rounding at the end. (qkv_norm_rope rounds after every module's output, as the module code it stands
// in for does; nothing else reads what this writes before the attention, so the intermediate roundings would only lose bits.)
// A group of D / 8 lanes owns one head's row, 16 bytes a lane. 8 192 rows (32 / 16 heads of 128, rotary, norms) 62.8 us, 270 MB read and
// written at 4.3 TB/s where a copy has 6.5: one token ahead in flight, a page's rows written by many SMs at different moments; one row each of 64 sequences 4.4 us, a launch and one chain of loads.
#include "common.cuh"
#include "host_util.h"
#include "paged.cuh"

namespace spinf {

struct AppendArgs {
  const __nv_bfloat16* qkv;
  int64_t pitch;
  int H, h;
  const __nv_bfloat16* wq;
  const __nv_bfloat16* wk;
  const __nv_bfloat16* cos_t;
  const __nv_bfloat16* sin_t;
  int half;  // rotary dimensions / 2 (0: none)
  float eps;
  int plus1, norm_v, skip_q;
  __nv_bfloat16* q_out;
  __nv_bfloat16* k_pages;
  __nv_bfloat16* v_pages;
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;
  int width;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = bf2_lo(w[i]), x[2 * i + 1] = bf2_hi(w[i]);
}

// A CTA walks tokens: 256 at a time it first works out where their rows go (a thread per token), then takes them one by one, all heads
// at once, four rows to a group of lanes; the next token's rows are on their way while this one's are worked on. The norm weights
// stay in registers, the rotary table is read once per token and lane.
template <int D>
__global__ void __launch_bounds__(256, 2) paged_append_kernel(const AppendArgs a, const PagedSeqs s, int* __restrict__ status) {
  constexpr int LANES = D / 8;         // lanes of a head's row
  constexpr int GROUPS = 256 / LANES;  // rows a CTA works on at once
  constexpr int RPT = 4;               // rows a group has in flight
  __shared__ int s_page[256], s_row[256];
  const int lane = threadIdx.x & 31, sub = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const uint32_t gmask = LANES == 32 ? 0xffffffffu : 0xffffu << (lane & 16);
  const int row0 = a.skip_q ? a.H : 0, rows = a.H + 2 * a.h - row0;
  const int blocks = (rows + GROUPS * RPT - 1) / (GROUPS * RPT);  // of rows a token makes
  const int hl = a.half / 8;  // lanes of a rotary half
  const int from = sub < hl ? sub + hl : sub < 2 * hl ? sub - hl : sub;
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
  if (a.wq) {
    wq = *reinterpret_cast<const uint4*>(a.wq + sub * 8);
    wk = *reinterpret_cast<const uint4*>(a.wk + sub * 8);
  }
  uint4 raw[RPT], cs = make_uint4(0, 0, 0, 0), sn = cs;
  auto fetch = [&](int64_t t, int blk) {
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = (blk * RPT + i) * GROUPS + group;
      if (r < rows) raw[i] = *reinterpret_cast<const uint4*>(a.qkv + t * a.pitch + static_cast<int64_t>(row0 + r) * D + sub * 8);
    }
    if (sub < 2 * hl) {
      const int64_t at = t * a.half + (sub < hl ? sub : sub - hl) * 8;
      cs = *reinterpret_cast<const uint4*>(a.cos_t + at);
      sn = *reinterpret_cast<const uint4*>(a.sin_t + at);
    }
  };
  for (int64_t t0 = blockIdx.x; t0 < s.n; t0 += 256ll * gridDim.x) {
    const int64_t left = (s.n - t0 + gridDim.x - 1) / gridDim.x;
    const int steps = static_cast<int>(left < 256 ? left : 256) * blocks;
    fetch(t0, 0);
    {
      const int64_t t = t0 + static_cast<int64_t>(threadIdx.x) * gridDim.x;
      int pg = -1, in_page = 0;
      if (t < s.n) {
        int lo = 0, hi = s.B;  // the row's sequence: how many sequences end at or before it
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (s.cu[mid + 1] <= t) lo = mid + 1;
          else hi = mid;
        }
        if (lo < s.B && t >= s.cu[lo]) {  // (a row behind the last sequence, or before the first, has no slot: its q is made, nothing else)
          const int slot = s.lens[lo] - s.cu[lo + 1] + static_cast<int>(t);
          in_page = slot & ((1 << s.page_log2) - 1);
          if (slot >= 0 && (slot >> s.page_log2) < a.width) pg = s.table[lo * s.table_pitch + (slot >> s.page_log2)];
          if (pg < 0 || pg >= s.n_pages) {
            pg = -1;
            atomicCAS(status, 0, ST_BAD_INDEX);
          }
        }
      }
      __syncthreads();  // the last 256 tokens' places have been read
      s_page[threadIdx.x] = pg;
      s_row[threadIdx.x] = in_page;
      __syncthreads();
    }
    int k = 0, blk = 0;
    for (int step = 0; step < steps; ++step) {
      const int64_t t = t0 + static_cast<int64_t>(k) * gridDim.x;
      const int pg = s_page[k], in_page = s_row[k], r0 = blk * RPT * GROUPS + group;
      uint4 cur[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) cur[i] = raw[i];
      float c[8], z[8];
      unpack8(cs, c);
      unpack8(sn, z);
      if (++blk == blocks) blk = 0, ++k;
      if (step + 1 < steps) fetch(t0 + static_cast<int64_t>(k) * gridDim.x, blk);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = r0 + i * GROUPS;
        if (r >= rows) continue;
        const int head = row0 + r;
        const bool is_q = head < a.H, is_v = head >= a.H + a.h;
        float x[8];
        unpack8(cur[i], x);
        if (is_v ? a.norm_v != 0 : a.wq != nullptr) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(gmask, ss, o, LANES);
          const float rs = rsqrtf(ss * (1.f / D) + a.eps);
          if (is_v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= rs;
          } else {
            float wf[8];
            unpack8(is_q ? wq : wk, wf);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * rs * (a.plus1 ? 1.f + wf[e] : wf[e]);
          }
        }
        if (a.half && !is_v) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(gmask, x[e], from, LANES);
          if (sub < 2 * hl) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = fmaf(x[e], c[e], (sub < hl ? -y[e] : y[e]) * z[e]);
          }
        }
        const uint4 packed = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
        if (is_q) {
          *reinterpret_cast<uint4*>(a.q_out + (t * a.H + head) * D + sub * 8) = packed;
        } else if (pg >= 0) {
          const int kh = head - a.H - (is_v ? a.h : 0);
          __nv_bfloat16* dst = is_v ? a.v_pages + pg * a.v_page + kh * a.v_head + in_page * a.v_row
                                    : a.k_pages + pg * a.k_page + kh * a.k_head + in_page * a.k_row;
          *reinterpret_cast<uint4*>(dst + sub * 8) = packed;
        }
      }
    }
  }
}

}  // namespace spinf

using namespace spinf;

extern "C" int spinf_paged_append(const void* qkv, int64_t pitch, int64_t n, int32_t H, int32_t Hkv, int32_t D, const void* wq,
                                  const void* wk, const void* cos_t, const void* sin_t, int32_t rot_dim, float eps, int32_t plus1,
                                  int32_t norm_v, void* q_out, void* k_pages, void* v_pages, int64_t n_pages, int32_t page,
                                  const int64_t* k_strides_host, const int64_t* v_strides_host, const int32_t* table,
                                  int64_t table_pitch, int32_t width, const int32_t* lens, const int32_t* cu, int32_t B, void* stream) {
  paged_launches = 0;
  if (n == 0 || (B == 0 && !q_out)) return 0;  // nothing to do: the row pointers may be null
  SPINF_CHECK_ARG(qkv && k_pages && v_pages && k_strides_host && v_strides_host && n > 0 && B >= 0);
  SPINF_CHECK_ARG(B == 0 || (table && lens && cu && width > 0 && table_pitch >= width));  // (no sequence: q's rows are made all the same)
  SPINF_CHECK_ARG(H > 0 && Hkv > 0 && (D == 128 || D == 256) && n < (1ll << 31) && pitch >= static_cast<int64_t>(H + 2 * Hkv) * D && pitch % 8 == 0);
  SPINF_CHECK_ARG(page >= 16 && page <= 256 && (page & (page - 1)) == 0 && n_pages > 0 && n_pages < (1ll << 31));
  SPINF_CHECK_ARG(static_cast<int64_t>(width) * page < (1ll << 31));
  SPINF_CHECK_ARG((wq != nullptr) == (wk != nullptr) && (cos_t != nullptr) == (sin_t != nullptr) && (cos_t != nullptr) == (rot_dim != 0));
  SPINF_CHECK_ARG(rot_dim >= 0 && rot_dim <= D && rot_dim % 16 == 0);
  SPINF_CHECK_ARG(q_out || (!wq && !cos_t));  // without norm and rotation q stays where it is
  if (B > PG_MAX_SEQS) return SPINF_ERR_TOO_LARGE;
  uintptr_t bits = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                   reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(wq) | reinterpret_cast<uintptr_t>(wk) |
                   reinterpret_cast<uintptr_t>(cos_t) | reinterpret_cast<uintptr_t>(sin_t);
  for (int i = 0; i < 3; ++i) bits |= static_cast<uintptr_t>(k_strides_host[i] | v_strides_host[i]) * 2;
  SPINF_CHECK_ARG((bits & 15) == 0);  // rows move 16 bytes at a time
  int dev = 0;
  SPINF_CUDA_OK(cudaGetDevice(&dev));
  int* status = status_word(dev);
  if (!status) return SPINF_ERR_CUDA;
  AppendArgs a;
  a.qkv = static_cast<const __nv_bfloat16*>(qkv);
  a.pitch = pitch;
  a.H = H;
  a.h = Hkv;
  a.wq = static_cast<const __nv_bfloat16*>(wq);
  a.wk = static_cast<const __nv_bfloat16*>(wk);
  a.cos_t = static_cast<const __nv_bfloat16*>(cos_t);
  a.sin_t = static_cast<const __nv_bfloat16*>(sin_t);
  a.half = rot_dim / 2;
  a.eps = eps;
  a.plus1 = plus1;
  a.norm_v = norm_v;
  a.skip_q = !q_out;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.k_pages = static_cast<__nv_bfloat16*>(k_pages);
  a.v_pages = static_cast<__nv_bfloat16*>(v_pages);
  a.k_page = k_strides_host[0], a.k_head = k_strides_host[1], a.k_row = k_strides_host[2];
  a.v_page = v_strides_host[0], a.v_head = v_strides_host[1], a.v_row = v_strides_host[2];
  a.width = width;
  PagedSeqs s = {};
  s.table = table;
  s.table_pitch = table_pitch;
  s.lens = lens;
  s.cu = cu;
  s.B = B;
  s.n_pages = static_cast<int>(n_pages);
  s.page_log2 = __builtin_ctz(static_cast<unsigned>(page));
  s.max_len = width * page;
  s.max_q = 0;  // the append sizes nothing by it
  s.n = n;
  const int64_t most = 2ll * sm_count();  // two CTAs an SM
  const int64_t grid = n < most ? n : most;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ++paged_launches;
  if (D == 256)
    paged_append_kernel<256><<<static_cast<unsigned>(grid), 256, 0, st>>>(a, s, status);
  else
    paged_append_kernel<128><<<static_cast<unsigned>(grid), 256, 0, st>>>(a, s, status);
  SPINF_CUDA_OK(cudaGetLastError());
  return 0;
}
