// A pool of cache pages as the host passes it, and its TMA tensor map.
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace spinf {

// a pool of pages as the host passes it
struct PagedPool {
  const void* base;
  int64_t n_pages, page, heads, dim;
  int64_t s_page, s_head, s_row;  // strides in elements
};
// tensor map over (64 dims, rows of a page, 64-dim slabs, heads, pages); one copy brings box_rows rows x box_slabs slabs of a head
int make_tmap_pages(CUtensorMap* out, const PagedPool& p, uint32_t box_rows, uint32_t box_slabs);


extern thread_local int64_t paged_launches;  // kernels that this thread's last paged call has launched

}  // namespace spinf
