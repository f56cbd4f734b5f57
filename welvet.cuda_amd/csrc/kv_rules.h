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

// Waves per SIMD that the attention kernels' registers leave room for, by
// head dims.
WV_HD constexpr int kv_waves(int hd) { return hd <= 64 ? 4 : hd <= 128 ? 3 : 2; }

// Capacity up to which every sequence is one part, so that nothing has to be
// joined: the more rows (K/V head and chunk of query heads of every sequence)
// there are, the less a cut is needed to fill the GPU, and the more bytes an
// entry's K and V have, the sooner it pays. A call's us whole and cut, of n
// sequences of an eighth of the capacity to all of it:
//   E4M3, 32 heads over 8 of 128 (256 bytes): 1 x 400 9.9 and 12.0, 1 x 600 10.9 and
//     12.3, 4 x 800 12.8 and 12.4, 16 x 800 12.8 and 15.3, 16 x 1500 18.3 and 15.5,
//     64 x 800 20.2 and 28.7, 64 x 2047 39.2 and 41.3, 256 x 4096 238 and 242
//   bf16, the same heads (512): 1 x 400 11.0 and 13.2, 16 x 800 15.6 and 17.1, 64 x 800
//     28.6 and 34.3, 64 x 2047 59.7 and 57.0
//   bf16, 12 over 4 of 64 (256): 1 x 600 9.0 and 11.5, 64 x 1200 14.7 and 19.0, 256 x
//     2400 71.2 and 67.3
//   fp32, 16 over 8 of 256 (2048): 1 x 400 36.2 and 29.8, 16 x 400 44.7 and 37.1, 64 x 1600
//     318 and 264, 256 x 1500 893 and 887
// The bound stays below where both meet at many rows, as one long sequence among
// short ones is then one workgroup's: 100 and one of 2047 among 64 34.7 whole, 20.2
// cut; 200 and one of 4096 among 256 91.3 and 68.8; among 1000, one of 8000 182 and
// 265, one of 16384 266 and 273. It goes by the capacity, as the host does not know
// the lengths: 256 of 125 to 1000 in a capacity of 4096 58 whole, 90 cut.
WV_HD int64_t kv_one_part(int64_t rows, int entry_bytes = 256) {
  const int64_t n = (650000 + 1350 * rows) / (512 + (entry_bytes > 256 ? entry_bytes : 256));
  return n > 256 ? n : 256;
}

// Workgroups of one wave instead of four, for many short sequences (whole ones:
// the bound is below kv_one_part's). The same heads: 130 of up to 64 9.9 us with one
// wave and 15.2 with four, up to 300 19.1 and 19.8, up to 800 36.9 and 32.1; 256 of
// up to 300 28.7 and 31.0, up to 800 56.8 and 50.2; 400 of up to 800 70.0 and 73.6, up
// to 2800 263 and 235; 1000 of up to 300 72.7 and 101.1, up to 1100 266 and 266; 256
// fp32 ones of up to 64, 16 heads over 8 of 256, 62.1 and 79.8.
WV_HD bool kv_one_wave(int64_t rows, int hd, int capacity) {
  return rows >= 200 * kv_waves(hd) && capacity <= rows / 4;
}

// Workgroups per row that fill 256 CUs once, and the tiles of `kt` entries
// that each takes of `tiles` (one at least per sequence): two for each of four
// waves, so that short sequences run side by side, or an equal share.
WV_HD int kv_target(int kv_rows, int hd) {
  const int n = 256 * kv_waves(hd) / kv_rows;
  return n > 1 ? n : 1;
}
constexpr int kKvLeastEntries = 256;
WV_HD int kv_part_tiles(int64_t tiles, int target, int kt) {
  const int64_t n = (tiles + target - 1) / target;
  return n > kKvLeastEntries / kt ? (int)n : kKvLeastEntries / kt;
}
// Longer shares are runs that go over the sequences' ends: 32 sequences of 512 to
// 4096 E4M3 entries, 32 heads over 8 of 128, 25 tiles each: 37.9 us with runs,
// 48.9 with parts; 64 of them up to 2000 40.5 and 46.1; 8 x 8192 in fp32, 16 heads
// of 64, 52.6 and 56.6.
WV_HD bool kv_runs(int64_t tiles, int target, int kt) {
  return kv_part_tiles(tiles, target, kt) > kKvLeastEntries / kt;
}
// Entries that a workgroup reads in the time that it takes to start another
// sequence of its run: 64 sequences of 512 to 4096 E4M3 entries, the kernel
// without the join, 67.9 us with 0, 62.9 with 128, 61.5 with 256, 62.5 with 512.
constexpr int kKvStart = 256;
// A sequence in runs: `start` units and its tiles (one where it has none).
WV_HD int kv_units(int tiles, int start) { return (tiles > 1 ? tiles : 1) + start; }
// What a run with `left` units to go has of the sequence that it meets at unit
// `off`: tiles [t0, t1), whether other runs have some before (index 0 or 1) and
// how many have one; left: the units for the sequences behind. false: it ends
// before the first tile, and the next run starts the sequence.
struct KvRun {
  int t0 = 0, t1 = 0, index = 0, parts = 1;
};
WV_HD bool kv_run(int tiles, int off, int start, int step, int& left, KvRun& r) {
  left -= off < start ? start - off : 0;
  if (left <= 0) return false;
  r.t0 = off < start ? 0 : off - start;
  const int behind = (tiles > 1 ? tiles : 1) - r.t0 - left;  // tiles for later runs
  r.t1 = r.t0 + left < tiles ? r.t0 + left : tiles;
  r.index = r.t0 > 0 ? 1 : 0;
  r.parts = r.t0 > 0 ? 2 : behind > 0 ? 1 + (behind + step - 1) / step : 1;
  left = behind < 0 ? -behind : 0;
  return true;
}
WV_HD int kv_parts(int tiles, int part_tiles) {
  const int n = (tiles + part_tiles - 1) / part_tiles;
  return n > 1 ? n : 1;
}
// Most workgroups of a row: full parts, and one that is not full per sequence;
// a sequence's parts hold kKvLeastEntries at least but for its last.
WV_HD int64_t kv_most_parts(int nseq, int target, int capacity) {
  const int64_t by_target = (int64_t)target + nseq;
  const int64_t by_capacity = (int64_t)nseq * ((capacity + kKvLeastEntries - 1) / kKvLeastEntries);
  return by_target < by_capacity ? by_target : by_capacity;
}
// How an attention call is cut, from what the host knows of it: sequences as
// long as they can be, `rows` of each (K/V heads and chunks of query heads); gen:
// ALiBi, windows or running sums. (The general kernels need more before runs pay
// for their longer prologue: 16 x 8191 entries with running sums, 12 heads over 4
// of 64, 26.2 us with runs, 25.5 with parts, 16 x 8192 of up to 3000 20.9 and 19.1;
// 32 x 8192 38.2 and 41.1.)
struct KvPlan {
  int target;     // kv_target; 0: every sequence is one part
  bool one, runs; // workgroups of one wave; kernels that may take runs
  int64_t parts;  // workgroups per row
};
WV_HD int kv_tile(int dtype) { return dtype == kKvF32 ? 16 : 32; }
WV_HD KvPlan kv_plan(int nseq, int rows, int hd, int capacity, int dtype, bool gen) {
  const int kt = kv_tile(dtype), target = kv_target(rows, hd);
  const int64_t all = (int64_t)nseq * rows, tiles = (int64_t)nseq * ((capacity + kt - 1) / kt);
  const bool whole = capacity <= kv_one_part(all, 2 * hd * kv_elem_bytes(dtype));
  KvPlan p;
  p.target = whole ? 0 : target;
  p.one = kv_one_wave(all, hd, capacity);
  p.runs = !whole && nseq > 1 && kv_runs(gen ? tiles / 2 : tiles, target, kt);
  p.parts = whole ? nseq : kv_most_parts(nseq, target, capacity);
  return p;
}
// Head dims that the attention kernel for `hd` is built for.
WV_HD int kv_padded_hd(int dtype, int hd) {
  if (dtype == kKvE4M3 || hd > 128) return (hd + 63) / 64 * 64;
  return (hd + 31) / 32 * 32;
}
// Most slots of a row for the sums of sequences of more than one part: two per
// run (the end of one sequence and the start of another); without runs, there
// are at most `target` full parts, and these sequences have one or more each.
WV_HD int64_t kv_most_slots(int target) { return 2 * (int64_t)target; }
// Where the sums of a sequence's parts are: part 0 in `slot`, part i > 0 in
// slot + 1 + (i - 1) stride.
struct KvInfo {
  int slot, parts, stride;
};
// As many of these parts as there are slots for. (All of them; but where lengths
// change during a call no workgroup may have said where a sequence's parts are,
// and what an earlier call left there, or zeros, is found.)
WV_HD KvInfo kv_held(KvInfo i, int slots) {
  if (i.slot < 0 || i.slot >= slots) i.slot = 0;
  i.stride = i.stride == 2 ? 2 : 1;
  const int behind = slots - 1 - i.slot;
  const int most = behind > 0 ? 2 + (behind - 1) / i.stride : 1;
  i.parts = i.parts < 1 ? 1 : i.parts < most ? i.parts : most;
  return i;
}

// First tile of `kt` entries that a window over indices leaves (0: no window).
WV_HD int kv_first_tile(int n, int qp, int window, int kt) {
  if (window <= 0 || qp < window) return 0;
  const int e = qp - window + 1;
  return (e < n ? e : n) / kt;
}

}  // namespace wv
