// Paged K/V cache for decoding: the pool, the calls' arguments and the kernel
// launchers (kvcache.hip).
#pragma once

#include "common.h"
#include "kv_rules.h"

namespace wv {

// The pool: K and V rows [num_pages][kv_heads][page_tokens][pitch] of dtype
// (elements hd .. pitch of a row are zero) and, for E4M3, one fp32 scale per
// row. Passed to kernels by value.
struct KvPool {
  uint8_t* k = nullptr;
  uint8_t* v = nullptr;
  float* ks = nullptr;
  float* vs = nullptr;
  int dtype = 0, num_pages = 0, page_tokens = 0, kv_heads = 0, heads = 0, hd = 0, pitch = 0;
  int max_pages = 0;
  WV_HD int capacity() const { return max_pages * page_tokens; }
  int64_t rows() const { return (int64_t)num_pages * kv_heads * page_tokens; }
};

// The sequences of a call (device pointers of the caller).
struct KvSeqs {
  int nseq = 0;
  const int32_t* table = nullptr;     // [nseq][max_pages]
  const int32_t* lens = nullptr;      // [nseq]
  const int32_t* next_pos = nullptr;  // [nseq], null: lens
  int32_t* pos = nullptr;             // [nseq][kv_heads][capacity], null: an entry's index
  float* weight = nullptr;            // [nseq][kv_heads][capacity], null: none
};

// A mounted cache: the pool and the scratch of the attention.
struct KvCache {
  KvPool pool;
  int max_seqs = 0;
  bool track = false;
  DevBuf k, v, ks, vs;
  DevBuf part, part_ml, info;  // KvPart::out, ml, info
  DevBuf scores, lse2;   // track: KvPart::scores and lse2
  // track, long capacities: the scratch of kv_choose (KvChooseLong)
  DevBuf choose_hist, choose_cut, choose_counts, choose_list;
};
Status kv_build(int dtype, int num_pages, int page_tokens, int heads, int kv_heads, int hd,
                int max_seqs, int max_pages, bool track, KvCache* c, hipStream_t st);

// k, v: fp32 rows of [kv_heads][hd], row b * rows + i at stride * (b * rows + i).
struct KvRows {
  int rows = 0;
  const int32_t* counts = nullptr;  // [nseq], null: rows
  const float* k = nullptr;
  const float* v = nullptr;
  int64_t k_stride = 0, v_stride = 0;
};
Status launch_kv_append(const KvPool& p, const KvSeqs& s, const KvRows& r, hipStream_t st);
// RoPE of one token per sequence at next_pos (lens without it): the pairs (d, d
// + hd / 2) of every head of q and k rows turned by next_pos / theta^(2 d / hd).
Status launch_kv_rope(float* q, float* k, int heads, int kv_heads, int hd, int q_stride,
                      int kv_stride, double theta, const KvPool& p, const KvSeqs& s, hipStream_t st);
Status launch_kv_read(const KvPool& p, const KvSeqs& s, int count, const int32_t* first,
                      const int32_t* counts, float* k, float* v, hipStream_t st);

struct KvAttend {
  const float* q = nullptr;  // row b: [heads][hd]
  float* out = nullptr;      // row b: [heads][hd]
  float* lse = nullptr;      // [nseq][heads] or null
  int64_t q_stride = 0, out_stride = 0;
  int tail = 0, window = 0, alibi = 0;
  float scale2 = 0.0f;  // scale * log2(e)
};
// How an attention call is cut, and its scratch. ml and out: per slot (a part
// of a sequence of more than one), row of query heads (K/V head and chunk of
// 16 heads) and head the reference and sum of the weights and the unscaled
// sums of V; scores (log2 units) and lse2: for the running sums, null without.
struct KvPart {
  int target = 0;             // kv_target; 0: every sequence is one part
  bool vec_q = false, vec_out = false;  // rows of q and out hold whole 16-byte pieces
  float* out = nullptr;       // [slots][rows][heads of a row][hd up to 4]
  float* ml = nullptr;        // [slots][rows][heads of a row][2]
  KvInfo* info = nullptr;     // [nseq], null where nothing follows the parts
  float* scores = nullptr;    // [nseq][heads][capacity]
  float* lse2 = nullptr;      // [nseq][heads]
};
Status kv_attend(const KvCache& c, const KvSeqs& s, const KvAttend& a, hipStream_t st);

Status kv_choose(const KvCache& c, const KvSeqs& s, int budget, int sinks, int recent, int32_t* src,
                 hipStream_t st);
Status launch_kv_compact(const KvPool& p, const KvSeqs& s, int budget, const int32_t* src,
                         hipStream_t st);
Status launch_kv_advance(int nseq, int32_t* lens, int32_t* next_pos, const int32_t* counts, int add,
                         int cap, hipStream_t st);

}  // namespace wv
