// A batch of requests as the kernels see it (gfx950), shared by the RoPE and attention kernels.
#pragma once

#include "common.h"

namespace llhip {
namespace {

constexpr int kMaxRequests = 1024; // LLHIP_MAX_REQUESTS

// Request r's rows, own length and slot; no rows (and bad set) where they leave the batch's buffers. A request without
// rows may hold anything else.
struct Request {
  int first, rows, length, slot;
};
__device__ __forceinline__ Request request_at(const RequestsDev &b, int r, bool &bad) {
  const int first = b.start[r], last = b.start[r + 1], length = b.length[r], slot = b.slot ? b.slot[r] : r;
  const bool rows_ok = first >= 0 && first <= last && last <= b.rows;
  const int n = rows_ok ? last - first : 0;
  const bool ok = rows_ok && (n == 0 || (length >= 0 && length <= b.seq_len - n && slot >= 0 && slot < b.slots));
  bad |= !ok;
  return Request{first, ok ? n : 0, length, slot};
}

} // namespace
} // namespace llhip
