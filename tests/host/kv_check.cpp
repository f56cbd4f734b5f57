// The K/V cache's index rules (csrc/kv_rules.h) behind a C interface.
#include "kv_rules.h"

extern "C" {

int kv_check_entries(int len, int tail, int cap) { return wv::kv_entries(len, tail, cap); }

long long kv_check_row(const int* table, int e, int h, int num_pages, int kv_heads, int page_tokens) {
  return wv::kv_row(table, e, h, num_pages, kv_heads, page_tokens);
}

int kv_check_pitch(int dtype, int hd) { return wv::kv_pitch(dtype, hd); }

float kv_check_scale(float amax) { return wv::kv_e4m3_scale(amax); }

unsigned kv_check_key(float w) { return wv::kv_weight_key(w); }

int kv_check_target(int rows, int hd) { return wv::kv_target(rows, hd); }

// Whether one-wave workgroups have only whole sequences.
int kv_check_one_wave(long long rows, int hd, int capacity) {
  return wv::kv_one_wave(rows, hd, capacity) ? 1 + (capacity <= wv::kv_one_part(rows)) : 0;
}

int kv_check_runs(long long tiles, int target, int kt) { return wv::kv_runs(tiles, target, kt) ? 1 : 0; }

int kv_check_part_tiles(long long tiles, int target, int kt) { return wv::kv_part_tiles(tiles, target, kt); }

int kv_check_parts(int tiles, int part_tiles) { return wv::kv_parts(tiles, part_tiles); }

long long kv_check_most_parts(int nseq, int target, int capacity) {
  return wv::kv_most_parts(nseq, target, capacity);
}

long long kv_check_most_slots(int target) { return wv::kv_most_slots(target); }

int kv_check_first_tile(int n, int qp, int window, int kt) { return wv::kv_first_tile(n, qp, window, kt); }

// Walks the runs of `step` units over sequences of tiles[b] tiles as the
// workgroups do: rows of {run, sequence, t0, t1, index, parts} in out (room for
// `most`); returns how many there are.
int kv_check_walk(const int* tiles, int nseq, int kt, int step, int* out, int most) {
  const int start = wv::kKvStart / kt;
  int rows = 0;
  long long total = 0;
  for (int b = 0; b < nseq; ++b) total += wv::kv_units(tiles[b], start);
  for (long long run = 0; run * step < total; ++run) {
    int b = 0, left = step;
    long long off = run * step;
    while (off >= wv::kv_units(tiles[b], start)) off -= wv::kv_units(tiles[b++], start);
    wv::KvRun r;
    while (wv::kv_run(tiles[b], (int)off, start, step, left, r)) {
      if (rows == most) return -1;
      int* o = out + 6 * rows++;
      o[0] = (int)run, o[1] = b, o[2] = r.t0, o[3] = r.t1, o[4] = r.index, o[5] = r.parts;
      if (left == 0 || ++b == nseq) break;
      off = 0;
      r = wv::KvRun();
    }
  }
  return rows;
}

int kv_check_start() { return wv::kKvStart; }

}  // extern "C"
