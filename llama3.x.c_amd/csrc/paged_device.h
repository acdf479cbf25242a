// A batch of requests over pages as the kernels see it (gfx950), shared by the append and attention kernels.
#pragma once

#include "common.h"

namespace llhip {
namespace {

constexpr int kMaxRequests = 1024; // LLHIP_MAX_REQUESTS

// Request r's rows and the positions before them; no rows (and bad set) where they leave the batch's buffers. A request
// without rows may hold anything else.
struct PagedRequest {
  int first, rows, length;
};
__device__ __forceinline__ PagedRequest paged_request(const PagedDev &b, int r, bool &bad) {
  const int first = b.start[r], last = b.start[r + 1], length = b.length[r];
  const bool rows_ok = first >= 0 && first <= last && last <= b.rows;
  const int n = rows_ok ? last - first : 0;
  const bool ok = rows_ok && (n == 0 || (length >= 0 && length <= b.seq_len - n));
  bad |= !ok;
  return PagedRequest{first, ok ? n : 0, length};
}

// The page that holds page_size positions of request r, number `i` of them, or -1 where it lies outside the caches.
__device__ __forceinline__ int page_of(const PagedDev &b, int r, int i) {
  const int page = b.pages[(size_t)r * b.max_pages + i];
  return (unsigned)page < (unsigned)b.num_pages ? page : -1;
}

} // namespace
} // namespace llhip
