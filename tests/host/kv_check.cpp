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

}  // extern "C"
