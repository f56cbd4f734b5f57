// Index rules of the paged K/V cache, for the host and the device: which
// entries a call covers and where an entry's row lies in the pool.
#pragma once

#include <stdint.h>

#include "codec.h"

namespace wv {

// Ids of the cache's element types (the reference's DType values).
enum KvType : int32_t { kKvF32 = 1, kKvBF16 = 3, kKvE4M3 = 4 };

constexpr int kKvMaxHd = 256;
// Pages hold whole groups of 16 entries: a matrix-core operand's rows.
constexpr int kKvGroup = 16;

WV_HD int kv_elem_bytes(int dtype) { return dtype == kKvF32 ? 4 : dtype == kKvBF16 ? 2 : 1; }

// Elements from an entry's row to the next one's: whole 16-byte pieces.
WV_HD int kv_pitch(int dtype, int hd) {
  const int n = 16 / kv_elem_bytes(dtype);
  return (hd + n - 1) / n * n;
}

// Entries of a sequence of `len` and `tail` more, within what a row of the
// page table covers; a negative length counts as none.
WV_HD int kv_entries(int len, int tail, int capacity) {
  if (len < 0) len = 0;
  if (len > capacity) len = capacity;
  return tail < capacity - len ? len + tail : capacity;
}

// Pool row of entry e: its page from the sequence's table row, -1 where that
// page is outside the pool (a hole: nothing is read or written there).
WV_HD int64_t kv_row(const int32_t* table_row, int e, int h, int num_pages, int kv_heads,
                     int page_tokens) {
  const int p = e / page_tokens;
  const int page = table_row[p];
  if (page < 0 || page >= num_pages) return -1;
  return ((int64_t)page * kv_heads + h) * page_tokens + (e - p * page_tokens);
}

// Scale of an E4M3 row with the largest magnitude amax: the weights' rule
// (scale_for), and at least 2^-96, so that a scale times a softmax weight of
// 24 bits stays a normal number. A row that holds inf or NaN (amax not finite)
// gets a scale of NaN: it reads back as NaN, not as the codes of finite values.
WV_HD float kv_e4m3_scale(float amax) {
  if (!(bits_of(amax) < 0x7F800000u)) return float_of(0x7FC00000u);
  const float s = scale_for(amax, max_representable(kE4M3));
  const float least = float_of((127u - 96u) << 23);
  return s < least ? least : s;
}

// Order of running sums: larger keys are kept first. NaN below everything.
WV_HD uint32_t kv_weight_key(float w) {
  const uint32_t u = bits_of(w);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
  // -inf maps to 0x007FFFFF, +inf to 0xFF800000; -0 counts as +0
  if (u == 0x80000000u) return 0x80000000u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t kKvKeyFirst = 0xFFFFFFFFu;  // sinks and recent entries

// Query heads of one K/V head are taken 16 at a time.
WV_HD int kv_chunks(int group) { return (group + 15) / 16; }

// Parts that the entries of every sequence are cut into at most, so that the
// attention's workgroups (4 waves of up to 256 registers: two per CU) fill 256
// CUs once; a part has at least 64 entries.
constexpr int kKvWorkgroups = 512;
WV_HD int kv_splits(int nseq, int kv_heads, int group, int capacity) {
  const int64_t rows = (int64_t)nseq * kv_heads * kv_chunks(group);
  int64_t n = kKvWorkgroups / rows;
  const int most = (capacity + 63) / 64;
  n = n < most ? n : most;
  return n > 1 ? (int)n : 1;
}

// A sequence's tiles of `kt` entries [first, end) and the tiles of each of its
// `parts`. window: of positions that are indices (0: none).
struct KvRange {
  int first, end, step, parts;
};
WV_HD KvRange kv_range(int n, int qp, int window, int kt, int splits) {
  KvRange r;
  r.end = (n + kt - 1) / kt;
  r.first = 0;
  if (window > 0 && qp >= window) {
    const int e = qp - window + 1;  // the first entry inside
    r.first = e / kt < r.end ? e / kt : r.end;
  }
  const int tiles = r.end - r.first;
  const int least = 64 / kt;
  r.step = (tiles + splits - 1) / splits;
  r.step = r.step < least ? least : r.step;
  r.parts = (tiles + r.step - 1) / r.step;
  return r;
}

}  // namespace wv
