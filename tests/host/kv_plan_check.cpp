// How the K/V cache's attention is cut (csrc/kv_rules.h) behind a C interface.
#include "kv_rules.h"

extern "C" {

// Bits: 1 whole sequences, 2 workgroups of one wave, 4 kernels that may take runs.
int kv_check_plan(int nseq, int rows, int hd, int capacity, int dtype, int gen) {
  const wv::KvPlan p = wv::kv_plan(nseq, rows, hd, capacity, dtype, gen != 0);
  return (p.target == 0 ? 1 : 0) | (p.one ? 2 : 0) | (p.runs ? 4 : 0);
}

int kv_check_padded_hd(int dtype, int hd) { return wv::kv_padded_hd(dtype, hd); }

// Whether the workgroups of a call over `tiles` take runs.
int kv_check_takes_runs(long long tiles, int rows, int hd, int dtype) {
  return wv::kv_runs(tiles, wv::kv_target(rows, hd), wv::kv_tile(dtype)) ? 1 : 0;
}

}  // extern "C"
