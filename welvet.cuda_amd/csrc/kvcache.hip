// Paged K/V cache for decoding: entries appended in the cache's type, the
// attention of one new token per sequence over them, and eviction by
// accumulated attention weight.
//
// Sequence b holds entries 0 .. len - 1; entry e lies in page table[b][e /
// page_tokens]. For query head j of K/V head h (j / (heads / kv_heads) = h)
//   s_e = scale q_j . k_e  (- slope_j |p_q - p_e| with ALiBi),
//   w_e = e^(s_e - lse),  lse = log(sum e^(s_e)),  out_j = sum w_e v_e
// over the entries that the window leaves (p_q - p_e < window); without any,
// out is 0 and lse -inf. Entries behind the length, in pages outside the pool
// and outside the window count as absent whatever their memory holds.
#include "kvcache.h"

#include "bf16.h"
#include "wave.h"

namespace wv {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f;

// ---------------------------------------------------------------------------
// Append: one group of lanes per (token, K/V head), four elements of its K
// and V rows per lane.
template <bool VEC>
__device__ __forceinline__ v4f load_row4(const float* row, int d, int hd) {
  v4f x = {0.f, 0.f, 0.f, 0.f};
  if constexpr (VEC) {
    if (d < hd) x = *reinterpret_cast<const v4f*>(row + d);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d + j < hd) x[j] = row[d + j];
  }
  return x;
}

// Two floats as bf16 (nearest, ties to even), the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)x, (__bf16)y});
}

// Canonical E4M3 code of x / s (encode_e4m3 of the rounded quotient) for |x| up
// to 240 s and y = 1 / s: the quotient x y corrected by the exact remainder
// is the correctly rounded one, without a division per element; half away from
// zero is the carry of an addition, and what lies below the least normal code
// (2^-6) is a signed zero. (2.7e8 quotients, next to ties and of any size,
// agreed with the division's; 8 x 512 tokens of 16 heads of 64: append 14.6 us
// with the division, 10.5 with this.)
__device__ __forceinline__ uint32_t e4m3_code(float x, float s, float y) {
  const float q0 = x * y;
  const float q = fmaf(fmaf(-q0, s, x), y, q0);
  const uint32_t a = bits_of(q) & 0x7FFFFFFFu;
  const uint32_t field = a < 0x3C800000u ? 0u : ((a + 0x80000u) >> 20) - (120u << 3);
  return (field & 0x7Fu) | (bits_of(q) >> 24 & 0x80u);
}

// Four elements of a row in the cache's type. Every lane of the group takes part
// (E4M3: in the row's maximum); those past the row (d >= pitch) store nothing.
__device__ __forceinline__ void store_row4(uint8_t* row, float* scale, v4f x, int dtype, int d,
                                           int pitch, int lanes) {
  if (dtype == kKvF32) {
    if (d < pitch) *reinterpret_cast<v4f*>(row + 4 * (size_t)d) = x;
  } else if (dtype == kKvBF16) {
    if (d < pitch)
      *reinterpret_cast<uint2*>(row + 2 * (size_t)d) =
          make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
  } else {
    // as integers: the order of magnitudes, with inf and NaN on top
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = bits_of(x[j]) & 0x7FFFFFFFu;
      m = u > m ? u : m;
    }
    for (int off = lanes / 2; off > 0; off >>= 1) {
      const uint32_t o = (uint32_t)__shfl_xor((int)m, off, 64);
      m = o > m ? o : m;
    }
    const float s = kv_e4m3_scale(float_of(m)), y = 1.0f / s;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= e4m3_code(x[j], s, y) << (8 * j);
    if (d < pitch) *reinterpret_cast<uint32_t*>(row + d) = w;
    if (d == 0) *scale = s;
  }
}

// A workgroup's groups of lanes over the rows of sequence blockIdx.y.
struct RowPlace {
  int b, j, h, d;  // sequence, token, K/V head, first element
  int64_t t;       // token row: b * rows + j
};
__device__ __forceinline__ bool row_place(const KvPool& p, int rows, int lanes, RowPlace& r) {
  const uint32_t i = (blockIdx.x * 256u + threadIdx.x) / (uint32_t)lanes;
  if (i >= (uint32_t)rows * (uint32_t)p.kv_heads) return false;
  r.b = blockIdx.y;
  r.j = (int)(i / (uint32_t)p.kv_heads);
  r.h = (int)(i - (uint32_t)r.j * (uint32_t)p.kv_heads);
  r.d = 4 * (threadIdx.x & (lanes - 1));
  r.t = (int64_t)r.b * rows + r.j;
  return true;
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void k_kv_append(KvPool p, KvSeqs s, KvRows r, int lanes) {
  RowPlace at;
  if (!row_place(p, r.rows, lanes, at)) return;
  if (r.counts && at.j >= r.counts[at.b]) return;
  const int cap = p.capacity(), h = at.h, d = at.d;
  const int len = s.lens[at.b];
  const int e = kv_entries(len, 0, cap) + at.j;
  if (e >= cap) return;
  const v4f kx = load_row4<VEC>(r.k + at.t * r.k_stride + (size_t)h * p.hd, d, p.hd);
  const v4f vx = load_row4<VEC>(r.v + at.t * r.v_stride + (size_t)h * p.hd, d, p.hd);
  const int64_t row = kv_row(s.table + (size_t)at.b * p.max_pages, e, h, p.num_pages, p.kv_heads,
                             p.page_tokens);
  if (d == 0) {
    const size_t i = ((size_t)at.b * p.kv_heads + h) * cap + e;
    if (s.pos) s.pos[i] = (s.next_pos ? s.next_pos[at.b] : len < 0 ? 0 : len) + at.j;
    if (s.weight) s.weight[i] = 0.0f;
  }
  if (row < 0) return;
  const size_t o = (size_t)row * p.pitch * kv_elem_bytes(DT);
  store_row4(p.k + o, p.ks + row, kx, DT, d, p.pitch, lanes);
  store_row4(p.v + o, p.vs + row, vx, DT, d, p.pitch, lanes);
}

// ---------------------------------------------------------------------------
// Read: entries first[b] + i as fp32, i < counts[b]; zero behind.
template <bool VEC>
__device__ __forceinline__ void write_row4(float* row, v4f x, int d, int hd) {
  if constexpr (VEC) {
    if (d < hd) *reinterpret_cast<v4f*>(row + d) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d + j < hd) row[d + j] = x[j];
  }
}

// Elements d .. d + 3 of a row (d a multiple of 4 below the pitch).
template <int DT>
__device__ __forceinline__ v4f read_row4(const uint8_t* row, int d) {
  if constexpr (DT == kKvF32) {
    return *reinterpret_cast<const v4f*>(row + 4 * (size_t)d);
  } else if constexpr (DT == kKvBF16) {
    const uint2 w = *reinterpret_cast<const uint2*>(row + 2 * (size_t)d);
    return v4f{float_of(w.x << 16), float_of(w.x & 0xFFFF0000u), float_of(w.y << 16),
               float_of(w.y & 0xFFFF0000u)};
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + d);
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return v4f{lo[0], lo[1], hi[0], hi[1]};
  }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void k_kv_read(KvPool p, KvSeqs s, int count,
                                                 const int32_t* __restrict__ first,
                                                 const int32_t* __restrict__ counts,
                                                 float* __restrict__ k, float* __restrict__ v,
                                                 int lanes) {
  RowPlace at;
  if (!row_place(p, count, lanes, at)) return;
  const int f = first ? first[at.b] : 0, c = counts ? counts[at.b] : count;
  v4f kx = {0.f, 0.f, 0.f, 0.f}, vx = kx;
  if (at.j < c && f >= 0 && f < p.capacity() - at.j) {
    const int64_t row = kv_row(s.table + (size_t)at.b * p.max_pages, f + at.j, at.h, p.num_pages,
                               p.kv_heads, p.page_tokens);
    if (row >= 0 && at.d < p.pitch) {
      const size_t o = (size_t)row * p.pitch * kv_elem_bytes(DT);
      kx = read_row4<DT>(p.k + o, at.d);
      vx = read_row4<DT>(p.v + o, at.d);
      if constexpr (DT == kKvE4M3) kx *= p.ks[row], vx *= p.vs[row];
    }
  }
  const size_t o = (at.t * p.kv_heads + at.h) * (size_t)p.hd;
  write_row4<VEC>(k + o, kx, at.d, p.hd);
  write_row4<VEC>(v + o, vx, at.d, p.hd);
}

// ---------------------------------------------------------------------------
// Attention of one new token. A workgroup of 4 waves takes the query heads of
// one K/V head (up to 16: the columns of a matrix-core tile) over one part of
// the entries, in tiles of 32 entries per wave (F32: 16):
//   S^T = K Q^T   K rows as they lie in the page are the A operand (lane 16 g
//                 + c: row c, 16 bytes from byte 64 i + 16 g), the queries
//                 the B operand. Lane 16 g + c ends with the scores of head c
//                 for entries 4 g + i of each group of 16;
//   O^T += V^T P^T  with those weights as the B operand where they are: the
//                 contraction runs over (g, i), so lane 16 g + c loads the V
//                 rows 4 g + i, dims c D .. c D + D - 1 (whole rows per 16
//                 lanes), and pairs of rows are interleaved in registers.
// Nothing goes through LDS until the waves' sums meet. BF16 and E4M3 entries
// (codes are exact in bf16) run on v_mfma_f32_16x16x32_bf16 with the queries
// and the weights in three bf16 terms each (2^-25 relative, so products of
// fp32 accuracy; one rounding to bf16 would leave 2^-9), F32 ones on
// v_mfma_f32_16x16x4_f32.
// The softmax is online in base 2. The reference of a head's weights moves
// only when a score exceeds it by more than kSlack (weights of up to 2^8 lose
// nothing in fp32), so most tiles need no exchange between lanes.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));

constexpr float kSlack = 8.0f;
constexpr int kKvFinishHeads = 64;  // heads whose sums k_kv_finish holds at once

// A piece of a V row. (Non-temporal: V lines are read whole by one instruction,
// and K lines by two, which keeps the ones of K in the caches between the two:
// 1 x 131072 entries of 8 heads of 128 in bf16 105.7 us with plain loads of
// both, 87.9 with these of V, 88.3 of K instead, 95.3 of both.)
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
  int i = 0;
#pragma unroll
  for (; i + 4 <= N; i += 4) {
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a4*>(p + 4 * i));
#pragma unroll
    for (int k = 0; k < 4; ++k) w[i + k] = x[k];
  }
  if constexpr (N % 4 >= 2) {
    const auto x = __builtin_nontemporal_load(reinterpret_cast<const u32x2_a4*>(p + 4 * (N / 4 * 4)));
    w[N / 4 * 4] = x[0], w[N / 4 * 4 + 1] = x[1];
  }
  if constexpr (N % 2 == 1) w[N - 1] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p + 4 * (N - 1)));
}

// Two E4M3 codes (the low or the high half of w) as two bf16.
template <bool HI>
__device__ __forceinline__ uint32_t cvt_e4m3(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
}

// Padded head dims of the kernels, and the next smaller one.
constexpr int kv_hd_below(int dtype, int hdp) {
  if (dtype == kKvE4M3) return hdp - 64;
  return hdp <= 128 ? hdp - 32 : hdp - 64;
}

template <int DT, int HDP>
struct KvShape {
  static constexpr int ELEM = DT == kKvF32 ? 4 : DT == kKvBF16 ? 2 : 1;
  static constexpr int NSUB = DT == kKvF32 ? 1 : 2;  // groups of 16 entries per tile
  static constexpr int KL = HDP * ELEM / 64;         // 16-byte loads of a K row per lane
  static constexpr int D = HDP / 16;                 // dims of V per lane
  static constexpr int VW = D * ELEM / 4;            // as dwords
  static constexpr int KS = HDP / 32;                // bf16 steps of a score
  // K loads that every head_dim of this kernel fills
  static constexpr int KFULL = (kv_hd_below(DT, HDP) * ELEM + 16) / 64;
};

// Sequence `b` of a call: entries, the query's position, the tiles to take.
template <int KT>
__device__ __forceinline__ void kv_sequence(const KvPool& p, const KvSeqs& s, const KvAttend& a, int b,
                                            int& n, int& qp, int& first, int& tiles) {
  const int len = s.lens[b];
  n = kv_entries(len, a.tail, p.capacity());
  qp = (s.next_pos ? s.next_pos[b] : kv_entries(len, 0, p.capacity())) + a.tail - 1;
  first = kv_first_tile(n, qp, s.pos == nullptr ? a.window : 0, KT);
  tiles = (n + KT - 1) / KT - first;
}

// x of the lane that a DPP control names, 0 where there is none.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int dpp_or_0(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}

// Inclusive sums over the lanes, by moves within rows of 16 and from the last
// lane of a row to the rows behind it (VALU operations, no LDS round trips).
__device__ __forceinline__ int wave_scan(int x) {
  x += dpp_or_0<0x111>(x);       // row_shr:1
  x += dpp_or_0<0x112>(x);       // row_shr:2
  x += dpp_or_0<0x114>(x);       // row_shr:4
  x += dpp_or_0<0x118>(x);       // row_shr:8
  x += dpp_or_0<0x142, 0xA>(x);  // row_bcast:15 to rows 1 and 3
  x += dpp_or_0<0x143, 0xC>(x);  // row_bcast:31 to rows 2 and 3
  return x;
}
__device__ __forceinline__ int wave_sum(int x) {
  return __builtin_amdgcn_readlane(wave_scan(x), 63);
}

// The tiles of workgroup blockIdx.x: [t0, t1) of sequence b, which has `parts`
// of them (index 0: its first), and where these are more than one the slot of
// its sums (KvInfo). Three ways to cut:
//   target 0: every sequence is one part;
//   parts of `step` tiles of one sequence each;
//   RUNS, many tiles: runs of `step` units over all sequences one after the
//   other, the same for every workgroup however unequal the sequences are (64
//   sequences of 512 to 4096 E4M3 entries, 32 heads over 8 of 128, whole calls:
//   parts 81.7 us, runs 75.7, and 69.0 since they count starts too: kv_units). A
//   workgroup ends one sequence, may take whole ones (left: its units still to
//   come) and starts another: two slots each.
struct KvPlace {
  int b, n, qp, t0, t1, index, parts, slot, stride, left, step;
};

// What a run has of sequence w.b from unit `off` on; false: none of its tiles.
template <int KT>
__device__ __forceinline__ bool kv_run_place(int first, int tiles, int off, KvPlace& w) {
  KvRun r;
  const bool has = kv_run(tiles, off, kKvStart / KT, w.step, w.left, r);
  w.t0 = first + r.t0, w.t1 = first + r.t1;
  w.index = r.index, w.parts = r.parts;
  w.slot = 2 * (int)blockIdx.x + (r.index > 0 ? 0 : 1);
  return has;
}

template <int KT, bool RUNS>
__device__ __forceinline__ bool kv_place(const KvPool& p, const KvSeqs& s, const KvAttend& a,
                                         const KvPart& part, int lane, KvPlace& w) {
  int first, tiles, index = 0;
  w.left = 0, w.stride = 1;
  if (s.nseq == 1 || part.target == 0) {
    w.b = s.nseq == 1 ? 0 : blockIdx.x;
    kv_sequence<KT>(p, s, a, w.b, w.n, w.qp, first, tiles);
    w.step = part.target == 0 ? tiles : kv_part_tiles(tiles, part.target, KT);
    w.parts = part.target == 0 ? 1 : kv_parts(tiles, w.step);
    index = s.nseq == 1 ? blockIdx.x : 0;
    w.slot = index;
    if (index >= w.parts) return false;
  } else {
    int n = 0, qp = 0, f = 0, t = 0;
    int64_t total = 0;
    for (int b0 = 0; b0 < s.nseq; b0 += 64) {
      t = 0;
      const bool in = b0 + lane < s.nseq;
      if (in) kv_sequence<KT>(p, s, a, b0 + lane, n, qp, f, t);
      // (halves, so that a wave's sum of up to 2^26 tiles each fits)
      const int units = in ? (t > 1 ? t : 1) : 0;
      total += wave_sum(units & 0xFFFF) + ((int64_t)wave_sum(units >> 16) << 16);
    }
    const bool runs = RUNS && kv_runs(total, part.target, KT);
    if (runs) total += (int64_t)s.nseq * (kKvStart / KT);
    w.step = kv_part_tiles(total, part.target, KT);
    const int64_t start = (int64_t)blockIdx.x * w.step;
    if (runs && start >= total) return false;
    int64_t units_before = 0;
    int parts_before = 0, slots_before = 0;
    unsigned long long hit = 0;
    for (int b0 = 0; b0 < s.nseq; b0 += 64) {
      const bool in = b0 + lane < s.nseq;
      if (s.nseq > 64 && in) kv_sequence<KT>(p, s, a, b0 + lane, n, qp, f, t);
      if (runs) {
        const int units = in ? kv_units(t, kKvStart / KT) : 0;
        const int64_t up = wave_scan(units & 0xFFFF) + ((int64_t)wave_scan(units >> 16) << 16);
        const int64_t at = start - units_before;
        hit = __ballot(in && at >= up - units && at < up);
        const int who = hit ? __builtin_ctzll(hit) : 63;
        // (what the lane before has)
        const int64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)up, who);
        const int64_t all = lo | ((int64_t)__builtin_amdgcn_readlane((int)(up >> 32), who) << 32);
        if (hit) index = (int)(at - (all - __builtin_amdgcn_readlane(units, who)));
        units_before += all;
      } else {
        const int parts = in ? kv_parts(t, w.step) : 0;
        const int up = wave_scan(parts);
        const unsigned long long ones = __ballot(parts == 1);  // (they take no slots)
        const int at = (int)blockIdx.x - parts_before;
        hit = __ballot(in && at >= up - parts && at < up);
        if (hit) {
          const int who = __builtin_ctzll(hit);
          w.parts = __builtin_amdgcn_readlane(parts, who);
          index = at - __builtin_amdgcn_readlane(up - parts, who);
          w.slot = slots_before + at - (int)__popcll(ones & ((1ull << who) - 1));
        }
        parts_before += __builtin_amdgcn_readlane(up, 63);
        slots_before += __builtin_amdgcn_readlane(up, 63) - (int)__popcll(ones);
      }
      if (hit) {
        const int who = __builtin_ctzll(hit);
        w.b = b0 + who;
        w.n = __builtin_amdgcn_readlane(n, who);
        w.qp = __builtin_amdgcn_readlane(qp, who);
        first = __builtin_amdgcn_readlane(f, who);
        tiles = __builtin_amdgcn_readlane(t, who);
        break;
      }
    }
    if (!hit) return false;
    if (runs) {
      w.left = w.step, w.stride = 2;
      return kv_run_place<KT>(first, tiles, index, w);
    }
  }
  w.index = index;
  w.t0 = first + index * w.step;
  w.t1 = w.t0 + w.step < first + tiles ? w.t0 + w.step : first + tiles;
  return true;
}

// The next sequence of a workgroup's run.
template <int KT>
__device__ __forceinline__ bool kv_next(const KvPool& p, const KvSeqs& s, const KvAttend& a, KvPlace& w) {
  if (w.left == 0 || w.b + 1 >= s.nseq) return false;
  ++w.b;
  int first, tiles;
  kv_sequence<KT>(p, s, a, w.b, w.n, w.qp, first, tiles);
  return kv_run_place<KT>(first, tiles, 0, w);
}

// GEN: ALiBi, windows, or scores for the running sums. RUNS: workgroups may take
// runs over several sequences. W waves per workgroup: 4, or 1 for many short
// sequences (kv_one_wave). Some RUNS kernels keep up to 20 registers in scratch
// (256 dims; general ones of 64 and 128) and are faster than parts all the same:
// 32 sequences of 512 to 4096, 16 heads over 8 of 256, fp32 297 us with runs and 410
// with parts, general 295 and 420, bf16 120 and 157, 128 and 166; 32 over 8 of 128,
// general, bf16 58.5 and 70.2, E4M3 42.5 and 55.5; 64 of 750 to 6000, E4M3, 16 over
// 8 of 64, 50.8 and 56.2, general 66 and 77, bf16, 12 over 4 of 64, general 45.8 and
// 52.8.
template <int DT, int HDP, bool GEN, bool RUNS, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(kv_waves(HDP), 8)))
void k_kv_attend(KvPool p, KvSeqs s, KvAttend a, KvPart part) {
  using T = KvShape<DT, HDP>;
  constexpr int NSUB = T::NSUB, KT = 16 * NSUB;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int group = p.heads / p.kv_heads, chunks = (group + 15) / 16;
  const int h = blockIdx.y / chunks, chunk = blockIdx.y % chunks;
  const int cols = group - 16 * chunk < 16 ? group - 16 * chunk : 16;
  const int head0 = h * group + 16 * chunk;
  const int cap = p.capacity();
  KvPlace place;
  if (!kv_place<KT, RUNS>(p, s, a, part, lane, place)) return;
  constexpr int STRIDE = HDP + 4;
  // one after the other: the queries' rows (16 rows of STRIDE floats), their
  // terms (F32: none, the rows stay), the waves' sums (a multiple of the rows)
  constexpr int QBYTES = DT == kKvF32 ? 0 : T::KS * 3 * 1024, SBYTES = W * 16 * STRIDE * 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[QBYTES > SBYTES ? QBYTES : SBYTES];
  static_assert(sizeof(lds) >= 16 * STRIDE * 4);
  __shared__ float ml[W][16][2];
  do {
    const int b = place.b, n = place.n, qp = place.qp, t0 = place.t0, t1 = place.t1;
    const int32_t* table = s.table + (size_t)b * p.max_pages;
    const int32_t* pos = s.pos ? s.pos + ((size_t)b * p.kv_heads + h) * cap : nullptr;

    const int row_bytes = p.pitch * T::ELEM;
    const int koff = c * row_bytes + 16 * g;
    // (dims behind the row: any valid address; they are not written out)
    const int vcol = c * T::D * T::ELEM < row_bytes ? c * T::D * T::ELEM : 0;
    const int voff = 4 * g * row_bytes + vcol;

    // Pages of this wave's tiles, 64 tiles at a time: lane i holds those of its
    // i-th tile from `from` on. (A load of its own for every tile would be waited
    // for at once, and with it, as loads return in order, all K and V loads.)
    int page[NSUB], at[NSUB];
    auto fetch = [&](int from) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        const int t = from + W * lane, e = t * KT + 16 * u;
        const int i = e / p.page_tokens;
        page[u] = t < t1 && e < n ? table[i] : -1;
        if (page[u] >= p.num_pages) page[u] = -1;
        at[u] = e - i * p.page_tokens;
      }
    };
    // pool rows of the groups of this wave's i-th tile; a group without entries
    // or page: -1
    auto rows_of = [&](int i, int64_t (&row)[NSUB]) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        const int pg = __builtin_amdgcn_readlane(page[u], i), off = __builtin_amdgcn_readlane(at[u], i);
        row[u] = pg >= 0 ? ((int64_t)pg * p.kv_heads + h) * p.page_tokens + off : -1;
      }
    };
    u32x4 kr[NSUB][T::KL];
    v4f ks[NSUB];
    auto load_k = [&](const int64_t (&row)[NSUB]) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        if constexpr (DT == kKvE4M3)
          ks[u] = *reinterpret_cast<const v4f*>(p.ks + (row[u] < 0 ? 0 : row[u]) + 4 * g);
        const uint8_t* base = p.k + (row[u] < 0 ? 0 : row[u]) * row_bytes;
#pragma unroll
        for (int i = 0; i < T::KL; ++i) {
          const bool in = i < T::KFULL || 64 * i + 16 * g < row_bytes;
          const u32x4 x = *reinterpret_cast<const u32x4*>(base + (in ? koff + 64 * i : 0));
          kr[u][i] = in ? x : u32x4{0, 0, 0, 0};
        }
      }
    };

    uint32_t vr[4 * NSUB][T::VW];
    v4f vs[NSUB];
    auto load_v = [&](const int64_t (&row)[NSUB]) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        const int64_t r = row[u] < 0 ? 0 : row[u];
        if constexpr (DT == kKvE4M3) vs[u] = *reinterpret_cast<const v4f*>(p.vs + r + 4 * g);
        const uint8_t* base = p.v + r * row_bytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<T::VW>(vr[4 * u + i], base + voff + i * row_bytes);
      }
    };

    int64_t row[NSUB], next[NSUB];
    int i = 0;  // of the tile in the pages held
    fetch(t0 + wave);
    rows_of(0, row);
    load_k(row);
    load_v(row);
    // queries: rows of heads in LDS with zeros around them, then this lane's part
    // of the contraction; the bf16 terms in LDS too, alike for the four waves
    const bool col_ok = c < cols;
    const float slope =
        GEN && a.alibi ? (float)(exp2(-8.0 * (double)(head0 + c + 1) / (double)p.heads) * kLog2e) : 0.0f;
    float* qrows = reinterpret_cast<float*>(lds);
    const float* q0 = a.q + (int64_t)b * a.q_stride + (int64_t)head0 * p.hd;
#pragma unroll
    for (int r = 0; r < (16 * HDP / 4 + 64 * W - 1) / (64 * W); ++r) {
      const int item = threadIdx.x + 64 * W * r, col = item / (HDP / 4), d = 4 * (item % (HDP / 4));
      v4f x = {0.f, 0.f, 0.f, 0.f};
      if (col < cols) {
        const float* from = q0 + col * p.hd + d;
        if (part.vec_q) {
          if (d < p.hd) x = *reinterpret_cast<const v4f*>(from);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (d + j < p.hd) x[j] = from[j];
        }
      }
      if (col < 16) *reinterpret_cast<v4f*>(qrows + col * STRIDE + d) = x;
    }
    __syncthreads();
    float mult = a.scale2;
    const float* qcol = qrows + c * STRIDE;
    if constexpr (DT != kKvF32) {
      float top = 0.0f;
      auto piece = [&](int step, int half) {
        const int d = DT == kKvBF16 ? 32 * step + 8 * g : 64 * (step / 2) + 16 * g + 8 * (step % 2);
        return *reinterpret_cast<const v4f*>(qcol + d + 4 * half);
      };
#pragma unroll
      for (int j = 0; j < 2 * T::KS; ++j) {
        const v4f x = piece(j / 2, j & 1);
        top = fmaxf(fmaxf(fmaxf(top, fabsf(x[0])), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      // terms of values of about 1: the third one of a small query would fall
      // below bf16's normal range
      int e = (int)(bits_of(top) >> 23) - 127;
      e = e < -126 || e > 126 ? 0 : e;
      mult *= pow2f(e);
      const float down = pow2f(-e);
      // this wave's steps, read before the terms take the rows' place
      constexpr int STEPS = (T::KS + W - 1) / W;
      v4f mine[STEPS][2];
#pragma unroll
      for (int r = 0; r < STEPS; ++r) {
        const int step = wave + W * r < T::KS ? wave + W * r : 0;
        mine[r][0] = piece(step, 0), mine[r][1] = piece(step, 1);
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < STEPS; ++r) {
        const int step = wave + W * r;
        if (step >= T::KS) break;
        bf16x8 qt[3];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          __bf16 t[3];
          split_bf16<3>(mine[r][j / 4][j % 4] * down, t);
#pragma unroll
          for (int k = 0; k < 3; ++k) qt[k][j] = t[k];
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)
          *reinterpret_cast<bf16x8*>(lds + (step * 3 + k) * 1024 + 16 * lane) = qt[k];
      }
      __syncthreads();
    }

    v4f acc[T::D];
#pragma unroll
    for (int d = 0; d < T::D; ++d) acc[d] = v4f{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;

    int qoff = DT == kKvF32 ? 4 * (c * STRIDE + 4 * g) : 16 * lane;
    for (int t = t0 + wave; t < t1; t += W) {
      // (the queries are read from LDS again for every tile: in registers they cost
      // a third of the waves)
      asm volatile("" : "+v"(qoff));
      if (++i == 64) {
        i = 0;
        fetch(t + W);
      }
      rows_of(i, next);
      // scores, the small terms apart from the large one
      v4f x[NSUB], small[NSUB];
#pragma unroll
      for (int u = 0; u < NSUB; ++u) x[u] = small[u] = v4f{0.f, 0.f, 0.f, 0.f};
      if constexpr (DT == kKvF32) {
#pragma unroll
        for (int i = 0; i < T::KL; ++i) {
          const v4f q = *reinterpret_cast<const v4f*>(lds + qoff + 64 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v4f& to = i & 1 ? small[0] : x[0];
            to = __builtin_amdgcn_mfma_f32_16x16x4f32(float_of(kr[0][i][j]), q[j], to, 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int step = 0; step < T::KS; ++step) {
          bf16x8 qt[3];
#pragma unroll
          for (int k = 0; k < 3; ++k)
            qt[k] = *reinterpret_cast<const bf16x8*>(lds + (step * 3 + k) * 1024 + qoff);
#pragma unroll
          for (int u = 0; u < NSUB; ++u) {
            bf16x8 k8;
            if constexpr (DT == kKvBF16) {
              k8 = __builtin_bit_cast(bf16x8, kr[u][step]);
            } else {
              const uint32_t w0 = kr[u][step / 2][2 * (step % 2)], w1 = kr[u][step / 2][2 * (step % 2) + 1];
              k8 = __builtin_bit_cast(bf16x8, u32x4{cvt_e4m3<false>(w0), cvt_e4m3<true>(w0),
                                                    cvt_e4m3<false>(w1), cvt_e4m3<true>(w1)});
            }
            small[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8, qt[2], small[u], 0, 0, 0);
            x[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8, qt[0], x[u], 0, 0, 0);
            small[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8, qt[1], small[u], 0, 0, 0);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        // (of an infinite K the query's first term has the sign; the others would
        // make it NaN or not as their signs and zeros fall)
        if constexpr (DT == kKvBF16) {
#pragma unroll
          for (int i = 0; i < 4; ++i) small[u][i] = __builtin_isinf(x[u][i]) ? 0.0f : small[u][i];
        }
        x[u] = (x[u] + small[u]) * mult;
        if constexpr (DT == kKvE4M3) x[u] *= ks[u];
      }
      const bool rows_ok = row[0] >= 0 && row[NSUB - 1] >= 0;
      const bool whole = rows_ok && (t + 1) * KT <= n && (!GEN || a.window <= 0);
      if (GEN && (a.alibi || a.window > 0)) {
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
          const int e = t * KT + 16 * u + 4 * g;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int ahead = qp - (pos ? pos[e + i < cap ? e + i : 0] : e + i);
            x[u][i] -= slope * fabsf((float)ahead);
            if (a.window > 0 && ahead >= a.window) x[u][i] = -INFINITY;
          }
        }
      }
      uint32_t unseen = 0;  // bit 4 u + i
      if (!whole) {
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = t * KT + 16 * u + 4 * g + i;
            bool seen = row[u] >= 0 && e < n;
            if (GEN && a.window > 0) seen = seen && qp - (pos ? pos[e < cap ? e : 0] : e) < a.window;
            if (!seen) x[u][i] = -INFINITY, unseen |= 1u << (4 * u + i);
          }
      }
      if (GEN && part.scores && col_ok) {
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
          const int e = t * KT + 16 * u + 4 * g;
          if (e < cap)  // (a capacity is whole groups of 16)
            *reinterpret_cast<v4f*>(part.scores + ((size_t)b * p.heads + head0 + c) * cap + e) = x[u];
        }
      }
      // (past the end: the pool's first rows; a branch around loads would make the
      // compiler wait for all of them where it ends)
      load_k(next);

      float top = x[0][0];
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, x[u][i]);
      if (__ballot(top > m + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float to = fmaxf(m, top);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= f;
#pragma unroll
        for (int d = 0; d < T::D; ++d) acc[d] *= f;
      }
      const float ref = m == -INFINITY ? 0.0f : m;
      float w[4 * NSUB];
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[4 * u + i] = __builtin_amdgcn_exp2f(x[u][i] - ref);
          l += w[4 * u + i];
        }
      // weights of 0 have to meet values that are finite
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 4 * NSUB; ++j)
          if (unseen >> j & 1) {
#pragma unroll
            for (int k = 0; k < T::VW; ++k) vr[j][k] = 0;
            if constexpr (DT == kKvE4M3) vs[j / 4][j % 4] = 0.0f;
          }
      }
      if constexpr (DT == kKvE4M3) {
#pragma unroll
        for (int j = 0; j < 4 * NSUB; ++j) w[j] *= vs[j / 4][j % 4];
      }
      if constexpr (DT == kKvF32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < T::D; ++d)
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(float_of(vr[i][d]), w[i], acc[d], 0, 0, 0);
      } else {
        // three terms of 8 bits each by cutting: they hold a weight's 24 exactly
        bf16x8 pt[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          u32x4 f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            f[j] = __builtin_amdgcn_perm(bits_of(w[2 * j + 1]), bits_of(w[2 * j]), 0x07060302u);
          pt[k] = __builtin_bit_cast(bf16x8, f);
          if (k < 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] -= float_of(bits_of(w[j]) & 0xFFFF0000u);
          }
        }
#pragma unroll
        for (int d = 0; d < T::D; ++d) {
          u32x4 f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (DT == kKvBF16) {
              f[j] = __builtin_amdgcn_perm(vr[2 * j + 1][d / 2], vr[2 * j][d / 2],
                                           d & 1 ? 0x07060302u : 0x05040100u);
            } else {
              const uint32_t two = __builtin_amdgcn_perm(vr[2 * j + 1][d / 4], vr[2 * j][d / 4],
                                                         d & 2 ? 0x07030602u : 0x05010400u);
              f[j] = d & 1 ? cvt_e4m3<true>(two) : cvt_e4m3<false>(two);
            }
          }
          const bf16x8 v8 = __builtin_bit_cast(bf16x8, f);
#pragma unroll
          for (int k = 2; k >= 0; --k)
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v8, pt[k], acc[d], 0, 0, 0);
        }
      }
      load_v(next);
#pragma unroll
      for (int u = 0; u < NSUB; ++u) row[u] = next[u];
    }

    // The waves' sums meet in LDS (over the queries' terms), then every thread
    // adds the four of its dims.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) ml[wave][c][0] = m, ml[wave][c][1] = l;
    __syncthreads();
    float* sums = reinterpret_cast<float*>(lds);
    if (col_ok) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) M = fmaxf(M, ml[w][c][0]);
      const float mine = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - M);
      float* to = sums + (wave * 16 + c) * STRIDE + 4 * g * T::D;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < T::D; ++d) to[i * T::D + d] = acc[d][i] * mine;
    }
    __syncthreads();
    if (part.info && place.index == 0 && blockIdx.y == 0 && threadIdx.x == 0)
      part.info[b] = KvInfo{place.slot, place.parts, place.stride};
    const bool one = place.parts == 1;
    const int most = group < 16 ? group : 16, pitch = (p.hd + 3) & ~3, quads = pitch / 4;
    // (lengths that change during the call can give slots past the last one)
    const int slot = (uint32_t)place.slot < (uint32_t)kv_most_slots(part.target) ? place.slot : 0;
    const size_t me = one ? 0 : ((size_t)slot * gridDim.y + blockIdx.y) * most;
    for (int item = threadIdx.x; item < cols * quads; item += 64 * W) {
      const int col = item / quads, quad = item - col * quads;
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) M = fmaxf(M, ml[w][col][0]);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float mw = ml[w][col][0];
        L += ml[w][col][1] * (mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - M));
      }
      v4f o = *reinterpret_cast<const v4f*>(sums + col * STRIDE + 4 * quad);
#pragma unroll
      for (int w = 1; w < W; ++w)
        o += *reinterpret_cast<const v4f*>(sums + (16 * w + col) * STRIDE + 4 * quad);
      if (!one) {  // this part's sums, for k_kv_finish
        if (quad == 0) part.ml[2 * (me + col)] = M, part.ml[2 * (me + col) + 1] = L;
        *reinterpret_cast<v4f*>(part.out + (me + col) * pitch + 4 * quad) = o;
        continue;
      }
      const size_t head = (size_t)b * p.heads + head0 + col;
      if (quad == 0) {
        const float lse2 = L == 0.0f ? -INFINITY : M + __builtin_amdgcn_logf(L);
        if (a.lse) a.lse[head] = lse2 * kLn2;
        if (part.lse2) part.lse2[head] = lse2;
      }
      o *= L == 0.0f ? 0.0f : 1.0f / L;
      float* out = a.out + (int64_t)b * a.out_stride + (int64_t)(head0 + col) * p.hd + 4 * quad;
      if (part.vec_out) {
        *reinterpret_cast<v4f*>(out) = o;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * quad + k < p.hd) out[k] = o[k];
      }
    }
    if constexpr (RUNS) __syncthreads();  // (the sums are read)
  } while (RUNS && kv_next<KT>(p, s, a, place));
}

template <class F>
__device__ __forceinline__ float over_lanes(float x, int lane, F&& f) {
  x = f(x, xor_lane<1>(x, lane));
  x = f(x, xor_lane<2>(x, lane));
  x = f(x, xor_lane<4>(x, lane));
  x = f(x, xor_lane<8>(x, lane));
  x = f(x, xor_lane<16>(x, lane));
  return f(x, xor_lane<32>(x, lane));
}

// Reference and sum of a head's weights over its parts, in every lane of the
// wave; at(i): where part i is.
template <class F>
__device__ __forceinline__ void join_sums(const float* ml, F&& at, int parts, int lane, float& top,
                                          float& sum) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  v2f mine = {-INFINITY, 0.0f};  // of the first 64
  if (lane < parts) mine = *reinterpret_cast<const v2f*>(ml + 2 * at(lane));
  top = mine[0];
  for (int i = lane + 64; i < parts; i += 64) top = fmaxf(top, ml[2 * at(i)]);
  top = over_lanes(top, lane, [](float x, float y) { return fmaxf(x, y); });
  auto part_sum = [&](float mi, float li) {
    return li * (mi == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mi - top));
  };
  sum = part_sum(mine[0], mine[1]);
  for (int i = lane + 64; i < parts; i += 64) sum += part_sum(ml[2 * at(i)], ml[2 * at(i) + 1]);
  sum = over_lanes(sum, lane, [](float x, float y) { return x + y; });
}

// What follows the parts, for sequence blockIdx.z and K/V head blockIdx.y:
// workgroups x < group join the parts of query head x (none where every
// sequence is one part); the others add the
// heads' weights to the running sums, 1024 entries at a time (the scores are
// there; a head's sum is formed again from its parts). A launch of its own, 4 to
// 6 us, costs no more than a join by the workgroup that is done last, whose
// parts have to pass the XCDs' L2: 24 x 1500 windowed E4M3 entries 14.7 us with
// the launch, 15.3 without it, 8 x 2047 in fp32 23.5 and 22.7, 16 x 8191 in bf16
// with running sums 25.3 and 27.7.
__global__ __launch_bounds__(256) void k_kv_finish(KvPool p, KvSeqs s, KvAttend a, KvPart part) {
  const int group = p.heads / p.kv_heads, chunks = kv_chunks(group);
  const int joins = part.target != 0 ? group : 0;
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int most = group < 16 ? group : 16, pitch = (p.hd + 3) & ~3;
  const size_t rows = (size_t)p.kv_heads * chunks;
  const KvInfo info = kv_held(part.info[b], (int)kv_most_slots(part.target));
  const int parts = info.parts;
  // part i of head j, counted in heads
  auto of = [&](int i, int j) {
    const size_t slot = (size_t)info.slot + (i ? 1 + (size_t)(i - 1) * info.stride : 0);
    return (slot * rows + (size_t)h * chunks + j / 16) * most + j % 16;
  };
  if ((int)blockIdx.x < joins) {
    if (parts == 1) return;  // written by the attention itself
    const int j = blockIdx.x;
    const size_t head = (size_t)b * p.heads + (size_t)h * group + j;
    // four dims per thread, several teams of threads over the parts; the first
    // four parts of a team are on their way while the references are reduced
    const int quads = pitch / 4, teams = 256 / quads;
    const int team = threadIdx.x / quads, quad = threadIdx.x - team * quads;
    constexpr int AHEAD = 4;
    v4f x[AHEAD];
    float mi[AHEAD];
    const int mine = team < teams ? parts : 0;
    auto load = [&](int i0) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int i = i0 + k * teams;
        const size_t at = of(i < parts ? i : i0, j);
        mi[k] = part.ml[2 * at];
        x[k] = *reinterpret_cast<const v4f*>(part.out + at * pitch + 4 * quad);
      }
    };
    if (team < mine) load(team);
    float top, sum;
    join_sums(part.ml, [&](int i) { return of(i, j); }, parts, lane, top, sum);
    v4f o = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = team; i0 < mine; i0 += AHEAD * teams) {
      if (i0 != team) load(i0);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (i0 + k * teams < parts)
          o += x[k] * (mi[k] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mi[k] - top));
    }
    __shared__ v4f meet[256];
    meet[threadIdx.x] = o;
    __syncthreads();
    if (team != 0) return;
    for (int k = 1; k < teams; ++k) o += meet[k * quads + quad];
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    float* out = a.out + (int64_t)b * a.out_stride + ((int64_t)h * group + j) * p.hd + 4 * quad;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (4 * quad + k < p.hd) out[k] = o[k] * f;
    if (a.lse && quad == 0)
      a.lse[head] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
    return;
  }
  int n, qp, first, tiles;
  kv_sequence<16>(p, s, a, b, n, qp, first, tiles);
  const int cap = p.capacity(), e0 = 16 * first + 1024 * ((int)blockIdx.x - joins);
  if (e0 >= n) return;
  const size_t head = (size_t)b * p.heads + (size_t)h * group;
  __shared__ float lse2[kKvFinishHeads];
  const float* sc = part.scores + head * cap;
  float* weight = s.weight + ((size_t)b * p.kv_heads + h) * cap;
  const int step = 1024 * ((int)gridDim.x - joins);
  for (int j0 = 0; j0 < group; j0 += kKvFinishHeads) {
    const int heads = group - j0 < kKvFinishHeads ? group - j0 : kKvFinishHeads;
    __syncthreads();
    for (int j = wave; j < heads; j += 4) {
      float x;
      if (parts == 1) {
        x = part.lse2[head + j0 + j];
      } else {
        float top, sum;
        join_sums(part.ml, [&](int i) { return of(i, j0 + j); }, parts, lane, top, sum);
        x = sum == 0.0f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
      }
      if (lane == 0) lse2[j] = x;
    }
    __syncthreads();
    for (int e = e0 + 4 * (int)threadIdx.x; e < n; e += step) {
      v4f w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int j = 0; j < heads; ++j) {
        const v4f x = *reinterpret_cast<const v4f*>(sc + (size_t)(j0 + j) * cap + e);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] += x[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[k] - lse2[j]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + k < n) weight[e + k] += w[k];
    }
  }
}

// ---------------------------------------------------------------------------
// Choice of the entries to keep, for one K/V head of one sequence: the key
// (kv_weight_key; sinks and recent entries on top) of the `budget`-th entry by
// counting the digits of the keys from the top (11, 11 and 10 bits), then the
// kept entries from behind the budget into the holes below it, both in index
// order. Counts are whole numbers, so the order in which lanes add them does
// not matter. Capacities of up to 16384 entries, with many rows 32768, take one
// workgroup and one launch, the keys held in registers; longer ones segments of
// 4096 entries with a workgroup each and a launch per step (k_kv_choose_long).
constexpr int kChooseThreads = 1024, kChooseWaves = kChooseThreads / 64;
constexpr int kChooseLong = 16 * kChooseThreads;  // more entries may be cut into segments
constexpr int kChooseOne = 32 * kChooseThreads;   // most entries of one workgroup
constexpr int kDigits = 2048;
constexpr int kShift[3] = {21, 10, 0};

// What is kept: keys above `least`, and the first `ties` entries at it.
struct KvCut {
  uint32_t least;
  int ties;
};

// The entries of a workgroup, whole runs of 64 per wave in index order.
template <int KPT>
struct KvKeys {
  uint32_t key[KPT];
  int first, end, runs;  // entry of run 0, lane 0 of this wave; the end of all; runs per wave

  __device__ __forceinline__ int entry(int i, int lane) const { return first + 64 * i + lane; }
  __device__ __forceinline__ void load(const KvPool& p, const KvSeqs& s, int b, int h, int sinks,
                                       int recent, int n, int from, int to, int wave, int lane) {
    const size_t base = ((size_t)b * p.kv_heads + h) * p.capacity();
    const float* weight = s.weight + base;
    const int32_t* pos = s.pos ? s.pos + base : nullptr;
    const int64_t late = (int64_t)(s.next_pos ? s.next_pos[b] : n) - recent;
    end = to;
    runs = (to - from + kChooseThreads - 1) / kChooseThreads;
    first = from + wave * runs * 64;
    // (every load from a valid address and without a branch around it: the
    // compiler would wait for each by itself; runs of no entries read the last)
    float w[KPT];
    int q[KPT];
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const int e = entry(i, lane);
      q[i] = e < end ? e : end - 1;
      w[i] = weight[q[i]];
    }
    if (pos) {
#pragma unroll
      for (int i = 0; i < KPT; ++i) q[i] = pos[q[i]];
    }
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      key[i] = q[i] < sinks || q[i] >= late ? kKvKeyFirst : kv_weight_key(w[i]);
  }
  // How many of this wave's entries lie below the budget.
  __device__ __forceinline__ int below(int budget) const {
    int last = first + 64 * runs < end ? first + 64 * runs : end;
    last = last < budget ? last : budget;
    return last > first ? last - first : 0;
  }
  // f(i, e, in): for every run, with all lanes
  template <class F>
  __device__ __forceinline__ void each(int lane, F&& f) const {
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      if (i < runs) f(i, entry(i, lane), entry(i, lane) < end);
  }
};

// Counts digit `step` of the keys that agree with `least` above it.
template <int KPT>
__device__ __forceinline__ void count_digits(const KvKeys<KPT>& keys, int step, uint32_t least,
                                             uint32_t* hist, int lane) {
  keys.each(lane, [&](int i, int, bool in) {
    const uint32_t k = keys.key[i];
    const bool on = in && (step == 0 || (k >> kShift[step - 1]) == (least >> kShift[step - 1]));
    const uint32_t digit = (k >> kShift[step]) & (step == 2 ? 1023u : 2047u);
    // the lanes that share the first one's digit add once (running sums of 0,
    // and entries that stay in any case, come in long runs)
    const unsigned long long act = __ballot(on);
    if (!act) return;
    const int lead = __builtin_ctzll(act);
    const uint32_t d0 = (uint32_t)__builtin_amdgcn_readlane((int)digit, lead);
    const unsigned long long same = __ballot(on && digit == d0);
    if (lane == lead) atomicAdd(&hist[d0], (uint32_t)__popcll(same));
    if (on && digit != d0) atomicAdd(&hist[digit], 1u);
  });
}

// Sum of the 16 waves' values before this one's; total: of all.
__device__ __forceinline__ int sum_before(const int* red, int wave, int lane, int& total) {
  static_assert(kChooseWaves == 16, "a row of 16 lanes holds the waves' values");
  const int up = wave_scan(red[lane & 15]);
  total = __builtin_amdgcn_readlane(up, 15);
  return wave ? __builtin_amdgcn_readlane(up, wave ? wave - 1 : 0) : 0;
}

// The digit of the need-th key from the top of hist (every thread calls);
// need becomes its rank among the keys of that digit. (0 and 0 where hist counts
// fewer: see KvList.)
__device__ __forceinline__ uint32_t find_digit(const uint32_t* hist, int& need, int* red, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  const int c0 = (int)hist[kDigits - 1 - 2 * tid], c1 = (int)hist[kDigits - 2 - 2 * tid];
  const int up = wave_scan(c0 + c1);
  if (lane == 63) red[wave] = up;
  if (tid == 0) red[kChooseWaves] = red[kChooseWaves + 1] = 0;
  __syncthreads();
  int all;
  const int before = up - c0 - c1 + sum_before(red, wave, lane, all);
  if (before < need && need <= before + c0 + c1) {
    const bool second = need > before + c0;
    red[kChooseWaves] = kDigits - 1 - 2 * tid - (second ? 1 : 0);
    red[kChooseWaves + 1] = need - before - (second ? c0 : 0);
  }
  __syncthreads();
  const uint32_t digit = (uint32_t)red[kChooseWaves];
  need = red[kChooseWaves + 1];
  __syncthreads();
  return digit;
}

// Sums over the earlier waves of one value per wave; total: of all.
__device__ __forceinline__ int waves_before(int x, int* red, int wave, int lane, int& total) {
  __syncthreads();
  if (lane == 0) red[wave] = x;
  __syncthreads();
  return sum_before(red, wave, lane, total);
}

// Entries at the cut, and above it, of a wave: below the budget and behind it.
struct KvCounts {
  int eq_low = 0, eq_high = 0, up_low = 0, up_high = 0;
};
template <int KPT>
__device__ __forceinline__ KvCounts count_cut(const KvKeys<KPT>& keys, uint32_t least, int budget,
                                              int lane) {
  KvCounts c;
  keys.each(lane, [&](int i, int e, bool in) {
    const bool eq = in && keys.key[i] == least, up = in && keys.key[i] > least;
    c.eq_low += __popcll(__ballot(eq && e < budget));
    c.eq_high += __popcll(__ballot(eq && e >= budget));
    c.up_low += __popcll(__ballot(up && e < budget));
    c.up_high += __popcll(__ballot(up && e >= budget));
  });
  return c;
}

// The kept entries from behind the budget: of n > budget entries, at most half
// move. Running sums, positions or lengths that are still being written while
// the call reads them several times can count more than there are: ranks past
// the list are dropped on both sides, so that such a call answers nothing but
// touches nothing outside its memory either.
struct KvList {
  int32_t* at;
  uint32_t room;
  __device__ __forceinline__ void put(int rank, int e) const {
    if ((uint32_t)rank < room) at[rank] = e;
  }
  // of what place_kept left in a slot: the entry of that hole
  __device__ __forceinline__ int take(int hole) const {
    const uint32_t rank = (uint32_t)(-2 - hole);
    return rank < room ? at[rank] : -1;
  }
};

// Writes the kept entries below the budget to src, the holes' ranks in their
// place (as -2 - rank), and the kept entries behind the budget to list. eq,
// holes, tails: how many come before this wave.
template <int KPT>
__device__ __forceinline__ void place_kept(const KvKeys<KPT>& keys, const KvCut& cut, int budget,
                                           int eq, int holes, int tails, int32_t* src, const KvList& list,
                                           int lane) {
  const unsigned long long before = (1ull << lane) - 1;
  keys.each(lane, [&](int i, int e, bool in) {
    const bool at = in && keys.key[i] == cut.least;
    const unsigned long long ats = __ballot(at);
    const bool kept = in && (keys.key[i] > cut.least || (at && eq + __popcll(ats & before) < cut.ties));
    eq += __popcll(ats);
    const bool low = in && e < budget;
    const unsigned long long hs = __ballot(low && !kept), ts = __ballot(in && !low && kept);
    if (low) src[e] = kept ? e : -2 - (holes + __popcll(hs & before));
    if (in && !low && kept) list.put(tails + __popcll(ts & before), e);
    holes += __popcll(hs);
    tails += __popcll(ts);
  });
}

// Kept entries at the cut among `eq` with `before` of them in front.
__device__ __forceinline__ int kept_at_cut(int ties, int before, int eq) {
  const int left = ties - before;
  return left < 0 ? 0 : left < eq ? left : eq;
}

template <int KPT>
__global__ __launch_bounds__(kChooseThreads) void k_kv_choose(KvPool p, KvSeqs s, int budget,
                                                              int sinks, int recent,
                                                              int32_t* __restrict__ out) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, cap = p.capacity();
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  __shared__ uint32_t hist[kDigits];
  __shared__ int red[kChooseWaves + 2];
  __shared__ int32_t tail[KPT * kChooseThreads / 2];
  const KvList list = {tail, KPT * kChooseThreads / 2};
  const int n = kv_entries(s.lens[b], 0, cap);
  int32_t* src = out + ((size_t)b * p.kv_heads + h) * budget;
  if (n <= budget) {
    for (int j = tid; j < budget; j += kChooseThreads) src[j] = j < n ? j : -1;
    return;
  }
  KvKeys<KPT> keys;
  keys.load(p, s, b, h, sinks, recent, n, 0, n, wave, lane);
  KvCut cut = {0u, budget};
#pragma unroll
  for (int step = 0; step < 3; ++step) {
    hist[tid] = 0, hist[tid + kChooseThreads] = 0;
    __syncthreads();
    count_digits(keys, step, cut.least, hist, lane);
    __syncthreads();
    cut.least |= find_digit(hist, cut.ties, red, tid) << kShift[step];
  }
  const KvCounts c = count_cut(keys, cut.least, budget, lane);
  int total;
  const int eq = waves_before(c.eq_low + c.eq_high, red, wave, lane, total);
  const int kept_low = c.up_low + kept_at_cut(cut.ties, eq, c.eq_low);
  const int kept_high = c.up_high + kept_at_cut(cut.ties, eq + c.eq_low, c.eq_high);
  const int low = keys.below(budget);
  const int holes = waves_before(low - kept_low, red, wave, lane, total);
  const int tails = waves_before(kept_high, red, wave, lane, total);
  place_kept(keys, cut, budget, eq, holes, tails, src, list, lane);
  __syncthreads();
  // (its own slots: every thread reads back what it wrote)
  keys.each(lane, [&](int, int e, bool) {
    const int at = e < budget ? src[e] : 0;
    if (at < -1) src[e] = list.take(at);
  });
}

// Long sequences: every step of the above a launch, a workgroup per segment of
// kSegment entries. The digits are counted in memory (zero between calls:
// k_kv_fill clears them), the ranks follow from the segments' counts. 2 x 8 rows of
// 100003 entries: 26 us in six launches of 2.0 to 7.0 us, of which each has about
// 2 us of launch and drain (the keys are 6.4 MB, read from the caches).
constexpr int kSegKeys = 4, kSegment = kSegKeys * kChooseThreads;

struct KvChooseLong {
  uint32_t* hist;    // [rows][3][kDigits]
  KvCut* cut;        // [rows][3]: after each digit
  KvCounts* counts;  // [rows][segments]
  int32_t* list;     // [rows][capacity / 2]
  int segments, budget, sinks, recent;
};

// STEP 0-2: count a digit; 3: count what is at and above the cut; 4: write
// the kept entries and list those behind the budget.
template <int STEP>
__global__ __launch_bounds__(kChooseThreads) void k_kv_choose_long(KvPool p, KvSeqs s, KvChooseLong c,
                                                                   int32_t* __restrict__ out) {
  const int h = blockIdx.y, b = blockIdx.z, seg = blockIdx.x, tid = threadIdx.x, cap = p.capacity();
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = b * p.kv_heads + h, budget = c.budget;
  __shared__ uint32_t hist[kDigits];
  __shared__ int red[kChooseWaves + 2];
  const int n = kv_entries(s.lens[b], 0, cap);
  int32_t* src = out + (size_t)row * budget;
  const int from = seg * kSegment, to = n - from < kSegment ? n : from + kSegment;
  if (n <= budget) {
    if (STEP == 4)
      for (int j = from + tid; j < budget && j < from + kSegment; j += kChooseThreads)
        src[j] = j < n ? j : -1;
    return;
  }
  if (from >= n) return;
  KvKeys<kSegKeys> keys;
  keys.load(p, s, b, h, c.sinks, c.recent, n, from, to, wave, lane);
  uint32_t* rows = c.hist + (size_t)row * 3 * kDigits;
  KvCut* cuts = c.cut + (size_t)row * 3;
  KvCut cut = {0u, budget};
  if constexpr (STEP >= 1) {
    if constexpr (STEP == 4) {
      cut = cuts[2];
    } else {
      if constexpr (STEP > 1) cut = cuts[STEP - 2];
      cut.least |= find_digit(rows + (STEP - 1) * kDigits, cut.ties, red, tid) << kShift[STEP - 1];
      if (seg == 0 && tid == 0) cuts[STEP - 1] = cut;
    }
  }
  if constexpr (STEP < 3) {
    hist[tid] = 0, hist[tid + kChooseThreads] = 0;
    __syncthreads();
    count_digits(keys, STEP, cut.least, hist, lane);
    __syncthreads();
    for (int i = tid; i < kDigits; i += kChooseThreads)
      if (hist[i]) atomicAdd(rows + STEP * kDigits + i, hist[i]);
    return;
  }
  KvCounts* counts = c.counts + (size_t)row * c.segments;
  const KvCounts w = count_cut(keys, cut.least, budget, lane);
  if constexpr (STEP == 3) {
    KvCounts all;
    waves_before(w.eq_low, red, wave, lane, all.eq_low);
    waves_before(w.eq_high, red, wave, lane, all.eq_high);
    waves_before(w.up_low, red, wave, lane, all.up_low);
    waves_before(w.up_high, red, wave, lane, all.up_high);
    if (tid == 0) counts[seg] = all;
  }
  if constexpr (STEP == 4) {
    // what lies in the segments before this one
    int eq0 = 0, holes0 = 0, tails0 = 0;
    for (int q0 = 0; q0 < seg; q0 += kChooseThreads) {
      const int q = q0 + tid;
      KvCounts x;
      if (q < seg) x = counts[q];
      const int eqs = x.eq_low + x.eq_high, up = wave_scan(eqs);
      int total, all;
      const int before = eq0 + waves_before(__builtin_amdgcn_readlane(up, 63), red, wave, lane, total) +
                         up - eqs;
      int low = budget - q * kSegment;
      low = q >= seg || low < 0 ? 0 : low < kSegment ? low : kSegment;
      const int hole = low - x.up_low - kept_at_cut(cut.ties, before, x.eq_low);
      const int tail = x.up_high + kept_at_cut(cut.ties, before + x.eq_low, x.eq_high);
      waves_before(wave_sum(q < seg ? hole : 0), red, wave, lane, all);
      holes0 += all;
      waves_before(wave_sum(q < seg ? tail : 0), red, wave, lane, all);
      tails0 += all;
      eq0 += total;
    }
    int total;
    const int eq = eq0 + waves_before(w.eq_low + w.eq_high, red, wave, lane, total);
    const int kept_low = w.up_low + kept_at_cut(cut.ties, eq, w.eq_low);
    const int kept_high = w.up_high + kept_at_cut(cut.ties, eq + w.eq_low, w.eq_high);
    const int low = keys.below(budget);
    const int holes = holes0 + waves_before(low - kept_low, red, wave, lane, total);
    const int tails = tails0 + waves_before(kept_high, red, wave, lane, total);
    const KvList list = {c.list + (size_t)row * (cap / 2), (uint32_t)cap / 2};
    place_kept(keys, cut, budget, eq, holes, tails, src, list, lane);
  }
}

// The last step: the holes (-2 - rank) take the listed entries, and the digits'
// counts, read no more, are cleared whatever the call found.
__global__ __launch_bounds__(256) void k_kv_fill(int budget, int half, int32_t* __restrict__ list,
                                                 uint32_t* __restrict__ hist, int32_t* __restrict__ out) {
  const size_t row = (size_t)blockIdx.z * gridDim.y + blockIdx.y;
  const int j = blockIdx.x * 256 + threadIdx.x;
  for (int i = j; i < 3 * kDigits; i += (int)gridDim.x * 256) hist[row * (3 * kDigits) + i] = 0;
  const KvList held = {list + row * half, (uint32_t)half};
  const int at = j < budget ? out[row * budget + j] : 0;
  if (at < -1) out[row * budget + j] = held.take(at);
}

// ---------------------------------------------------------------------------
// Compaction: a wave looks at 64 slots and moves the rows of those that get
// another entry, as many rows at a time as 64 lanes of 16 bytes hold. Sources
// lie behind the budget and targets below it, so the order is free.
template <int LANES>  // per row
__global__ __launch_bounds__(256) void k_kv_compact(KvPool p, KvSeqs s, int budget,
                                                    const int32_t* __restrict__ src) {
  const int lane = threadIdx.x & 63, h = blockIdx.y, b = blockIdx.z, cap = p.capacity();
  const int j = blockIdx.x * 256 + threadIdx.x;
  const size_t row = (size_t)b * p.kv_heads + h;
  const int e = j < budget ? src[row * budget + j] : -1;
  const bool move = e >= budget && e < cap;  // (otherwise its own, none, or outside)
  int64_t from = -1, to = -1;
  if (move) {
    const int32_t* table = s.table + (size_t)b * p.max_pages;
    from = kv_row(table, e, h, p.num_pages, p.kv_heads, p.page_tokens);
    to = kv_row(table, j, h, p.num_pages, p.kv_heads, p.page_tokens);
    // (an entry in a hole has no K and V to move: the slot keeps its own whole)
    if (s.weight && from >= 0) s.weight[row * cap + j] = s.weight[row * cap + e];
    if (s.pos && from >= 0) s.pos[row * cap + j] = s.pos[row * cap + e];
  }
  const bool on = from >= 0 && to >= 0;
  const unsigned long long mask = __ballot(on);
  const int count = __popcll(mask);
  if (count == 0) return;
  if (on && p.dtype == kKvE4M3) p.ks[to] = p.ks[from], p.vs[to] = p.vs[from];
  // the k-th move's rows to lane k: a permutation of the lanes
  const int below = __popcll(mask & ((1ull << lane) - 1));
  const int at = 4 * (on ? below : count + lane - below);
  const int from_lo = __builtin_amdgcn_ds_permute(at, (int)from), from_hi = __builtin_amdgcn_ds_permute(at, (int)(from >> 32));
  const int to_lo = __builtin_amdgcn_ds_permute(at, (int)to), to_hi = __builtin_amdgcn_ds_permute(at, (int)(to >> 32));
  const int bytes = p.pitch * kv_elem_bytes(p.dtype);
  constexpr int TEAMS = 64 / LANES, AHEAD = 4;
  const int team = lane / LANES, o = 16 * (lane % LANES);
  for (int k0 = 0; k0 < count; k0 += TEAMS * AHEAD) {
    v4f kx[AHEAD], vx[AHEAD];
    int64_t dst[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = k0 + u * TEAMS + team, who = k < 64 ? k : 63;
      const int64_t f = ((int64_t)__shfl(from_hi, who, 64) << 32) | (uint32_t)__shfl(from_lo, who, 64);
      const int64_t t = ((int64_t)__shfl(to_hi, who, 64) << 32) | (uint32_t)__shfl(to_lo, who, 64);
      dst[u] = k < count && o < bytes ? t * bytes + o : -1;
      if (dst[u] >= 0) {
        kx[u] = *reinterpret_cast<const v4f*>(p.k + f * bytes + o);
        vx[u] = *reinterpret_cast<const v4f*>(p.v + f * bytes + o);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (dst[u] >= 0) {
        *reinterpret_cast<v4f*>(p.k + dst[u]) = kx[u];
        *reinterpret_cast<v4f*>(p.v + dst[u]) = vx[u];
      }
  }
}

// ---------------------------------------------------------------------------
// RoPE of one token per sequence (launch_kv_rope), in f64 as the attention
// layers' own (k_rope): a workgroup per sequence forms the angles once for all
// heads.
__global__ __launch_bounds__(256) void k_kv_rope(float* __restrict__ q, float* __restrict__ k,
                                                 int heads, int kv_heads, int hd, int q_stride,
                                                 int kv_stride, double theta, KvPool p, KvSeqs s) {
  const int b = blockIdx.x, half = hd / 2;
  __shared__ double cs[kKvMaxHd / 2][2];
  const int t = s.next_pos ? s.next_pos[b] : kv_entries(s.lens[b], 0, p.capacity());
  for (int d = threadIdx.x; d < half; d += 256) {
    const double ang = (double)t / pow(theta, (double)(2 * d) / (double)hd);
    cs[d][0] = cos(ang), cs[d][1] = sin(ang);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < (heads + kv_heads) * half; i += 256) {
    const int h = i / half, d = i - h * half;
    float* row = h < heads ? q + (size_t)b * q_stride + (size_t)h * hd
                           : k + (size_t)b * kv_stride + (size_t)(h - heads) * hd;
    const double c = cs[d][0], n = cs[d][1], a0 = row[d], a1 = row[d + half];
    row[d] = (float)(a0 * c - a1 * n);
    row[d + half] = (float)(a0 * n + a1 * c);
  }
}

__global__ void k_kv_advance(int nseq, int32_t* lens, int32_t* next_pos,
                             const int32_t* __restrict__ counts, int add, int cap) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= nseq) return;
  int c = counts ? counts[b] : add;
  c = c < 0 ? 0 : c > add ? add : c;
  lens[b] = kv_entries(lens[b], c, cap);
  if (next_pos) next_pos[b] += c;
}

int64_t blocks_of(int64_t threads) { return (threads + 255) / 256; }

}  // namespace

Status kv_build(int dtype, int num_pages, int page_tokens, int heads, int kv_heads, int hd,
                int max_seqs, int max_pages, bool track, KvCache* c, hipStream_t st) {
  KvPool& p = c->pool;
  p.dtype = dtype, p.num_pages = num_pages, p.page_tokens = page_tokens, p.heads = heads;
  p.kv_heads = kv_heads, p.hd = hd, p.pitch = kv_pitch(dtype, hd), p.max_pages = max_pages;
  c->max_seqs = max_seqs, c->track = track;
  const size_t rows = (size_t)p.rows();
  const size_t bytes = rows * p.pitch * kv_elem_bytes(dtype);
  for (DevBuf* b : {&c->k, &c->v}) {
    // (256 bytes more: a lane's piece of the last V row may end behind it)
    WV_TRY(b->alloc(bytes + 256));
    WV_HIP(hipMemsetAsync(b->p, 0, bytes + 256, st));
  }
  if (dtype == kKvE4M3)
    for (DevBuf* b : {&c->ks, &c->vs}) {
      WV_TRY(b->alloc(rows * sizeof(float)));
      WV_HIP(hipMemsetAsync(b->p, 0, rows * sizeof(float), st));
    }
  if (track) {
    WV_TRY(c->scores.alloc((size_t)max_seqs * heads * p.capacity() * sizeof(float)));
    WV_TRY(c->lse2.alloc((size_t)max_seqs * heads * sizeof(float)));
  }
  const int chunk_rows = kv_heads * kv_chunks(heads / kv_heads);
  const int most = heads / kv_heads < 16 ? heads / kv_heads : 16;
  const size_t slots = (size_t)kv_most_slots(kv_target(chunk_rows, hd)) * chunk_rows * most;
  WV_TRY(c->part.alloc(slots * ((hd + 3) & ~3) * sizeof(float)));
  WV_TRY(c->part_ml.alloc(slots * 2 * sizeof(float)));
  WV_TRY(c->info.alloc((size_t)max_seqs * sizeof(KvInfo)));
  WV_HIP(hipMemsetAsync(c->info.p, 0, c->info.bytes, st));
  if (track && p.capacity() > kChooseLong) {
    const size_t choose_rows = (size_t)max_seqs * kv_heads;
    WV_TRY(c->choose_hist.alloc(choose_rows * 3 * kDigits * sizeof(uint32_t)));
    WV_HIP(hipMemsetAsync(c->choose_hist.p, 0, c->choose_hist.bytes, st));
    WV_TRY(c->choose_cut.alloc(choose_rows * 3 * sizeof(KvCut)));
    const size_t segments = (p.capacity() + kSegment - 1) / kSegment;
    WV_TRY(c->choose_counts.alloc(choose_rows * segments * sizeof(KvCounts)));
    WV_TRY(c->choose_list.alloc(choose_rows * (p.capacity() / 2) * sizeof(int32_t)));
  }
  WV_HIP(hipStreamSynchronize(st));
  p.k = c->k.as<uint8_t>(), p.v = c->v.as<uint8_t>();
  p.ks = c->ks.as<float>(), p.vs = c->vs.as<float>();
  return Status::ok();
}

// Lanes that take a row, four elements each, and the grid over the rows of
// every sequence.
int row_lanes(const KvPool& p) {
  int lanes = 1;
  while (4 * lanes < p.pitch) lanes *= 2;
  return lanes;
}
Status row_grid(const KvPool& p, int nseq, int rows, int lanes, dim3* grid) {
  const int64_t threads = (int64_t)rows * p.kv_heads * lanes;
  if (threads > INT32_MAX)
    return Status::err(kInvalid, "kv: rows * num_kv_heads * head_dim of one sequence too large");
  *grid = dim3((unsigned)blocks_of(threads), (unsigned)nseq);
  return Status::ok();
}

template <int DT>
void append_of(bool vec, dim3 grid, const KvPool& p, const KvSeqs& s, const KvRows& r, int lanes,
               hipStream_t st) {
  if (vec)
    k_kv_append<DT, true><<<grid, 256, 0, st>>>(p, s, r, lanes);
  else
    k_kv_append<DT, false><<<grid, 256, 0, st>>>(p, s, r, lanes);
}

Status launch_kv_append(const KvPool& p, const KvSeqs& s, const KvRows& r, hipStream_t st) {
  if (s.nseq == 0 || r.rows == 0) return Status::ok();
  const int lanes = row_lanes(p);
  dim3 grid;
  WV_TRY(row_grid(p, s.nseq, r.rows, lanes, &grid));
  const bool vec = p.hd % 4 == 0 && r.k_stride % 4 == 0 && r.v_stride % 4 == 0 &&
                   ((uintptr_t)r.k | (uintptr_t)r.v) % 16 == 0;
  if (p.dtype == kKvF32) append_of<kKvF32>(vec, grid, p, s, r, lanes, st);
  else if (p.dtype == kKvBF16) append_of<kKvBF16>(vec, grid, p, s, r, lanes, st);
  else append_of<kKvE4M3>(vec, grid, p, s, r, lanes, st);
  return hip_status(hipGetLastError(), "k_kv_append");
}

template <int DT>
void read_of(bool vec, dim3 grid, const KvPool& p, const KvSeqs& s, int count, const int32_t* first,
             const int32_t* counts, float* k, float* v, int lanes, hipStream_t st) {
  if (vec)
    k_kv_read<DT, true><<<grid, 256, 0, st>>>(p, s, count, first, counts, k, v, lanes);
  else
    k_kv_read<DT, false><<<grid, 256, 0, st>>>(p, s, count, first, counts, k, v, lanes);
}

Status launch_kv_read(const KvPool& p, const KvSeqs& s, int count, const int32_t* first,
                      const int32_t* counts, float* k, float* v, hipStream_t st) {
  if (s.nseq == 0 || count == 0) return Status::ok();
  const int lanes = row_lanes(p);
  dim3 grid;
  WV_TRY(row_grid(p, s.nseq, count, lanes, &grid));
  const bool vec = p.hd % 4 == 0 && ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
  if (p.dtype == kKvF32) read_of<kKvF32>(vec, grid, p, s, count, first, counts, k, v, lanes, st);
  else if (p.dtype == kKvBF16) read_of<kKvBF16>(vec, grid, p, s, count, first, counts, k, v, lanes, st);
  else read_of<kKvE4M3>(vec, grid, p, s, count, first, counts, k, v, lanes, st);
  return hip_status(hipGetLastError(), "k_kv_read");
}

template <int DT>
Status launch_attend(int hd, bool one, bool gen, bool runs, dim3 grid, const KvPool& p, const KvSeqs& s,
                     const KvAttend& a, const KvPart& part, hipStream_t st) {
#define WV_KV_HD(N)                                                                     \
  (one && gen ? k_kv_attend<DT, N, true, false, 1><<<grid, 64, 0, st>>>(p, s, a, part)    \
   : one      ? k_kv_attend<DT, N, false, false, 1><<<grid, 64, 0, st>>>(p, s, a, part)   \
   : gen && runs ? k_kv_attend<DT, N, true, true, 4><<<grid, 256, 0, st>>>(p, s, a, part)    \
   : gen      ? k_kv_attend<DT, N, true, false, 4><<<grid, 256, 0, st>>>(p, s, a, part)   \
   : runs     ? k_kv_attend<DT, N, false, true, 4><<<grid, 256, 0, st>>>(p, s, a, part)   \
              : k_kv_attend<DT, N, false, false, 4><<<grid, 256, 0, st>>>(p, s, a, part))
  const int padded = kv_padded_hd(DT, hd);
  if constexpr (DT != kKvE4M3) {
    if (padded == 32) WV_KV_HD(32);
    else if (padded == 96) WV_KV_HD(96);
  }
  if (padded == 64) WV_KV_HD(64);
  else if (padded == 128) WV_KV_HD(128);
  else if (padded == 192) WV_KV_HD(192);
  else if (padded == 256) WV_KV_HD(256);
#undef WV_KV_HD
  return hip_status(hipGetLastError(), "k_kv_attend");
}

Status kv_attend(const KvCache& c, const KvSeqs& s, const KvAttend& a, hipStream_t st) {
  if (s.nseq == 0) return Status::ok();
  const KvPool& p = c.pool;
  const int rows = p.kv_heads * kv_chunks(p.heads / p.kv_heads);
  KvPart part;
  const bool gen = a.alibi || a.window > 0 || s.weight;
  const KvPlan plan = kv_plan(s.nseq, rows, p.hd, p.capacity(), p.dtype, gen);
  part.target = plan.target;
  part.out = c.part.as<float>();
  part.ml = c.part_ml.as<float>();
  part.vec_q = p.hd % 4 == 0 && a.q_stride % 4 == 0 && (uintptr_t)a.q % 16 == 0;
  part.vec_out = p.hd % 4 == 0 && a.out_stride % 4 == 0 && (uintptr_t)a.out % 16 == 0;
  const bool finish = part.target != 0 || s.weight;
  if (finish) part.info = c.info.as<KvInfo>();
  if (s.weight) {
    part.scores = c.scores.as<float>();
    part.lse2 = c.lse2.as<float>();
  }
  const dim3 grid((unsigned)plan.parts, (unsigned)rows);
  WV_TRY(p.dtype == kKvF32    ? launch_attend<kKvF32>(p.hd, plan.one, gen, plan.runs, grid, p, s, a, part, st)
         : p.dtype == kKvBF16 ? launch_attend<kKvBF16>(p.hd, plan.one, gen, plan.runs, grid, p, s, a, part, st)
                              : launch_attend<kKvE4M3>(p.hd, plan.one, gen, plan.runs, grid, p, s, a, part, st));
  if (!finish) return Status::ok();
  const int most = (p.capacity() + 1023) / 1024;
  const int track = !s.weight ? 0 : most < 64 ? most : 64;
  const int joins = part.target != 0 ? p.heads / p.kv_heads : 0;
  k_kv_finish<<<dim3(joins + track, p.kv_heads, s.nseq), 256, 0, st>>>(p, s, a, part);
  return hip_status(hipGetLastError(), "k_kv_finish");
}

Status kv_choose(const KvCache& c, const KvSeqs& s, int budget, int sinks, int recent, int32_t* src,
                 hipStream_t st) {
  if (s.nseq == 0) return Status::ok();
  const KvPool& p = c.pool;
  const dim3 grid(p.kv_heads, s.nseq);
  const int cap = p.capacity();
  // (up to kChooseOne, rows enough keep the GPU busy with a workgroup each: 8 x 20000
  // entries of 8 heads 31.2 us so and 26.4 in segments, 32 x 20000 31.9 and 53.9; 8 x
  // 32000 42.6 and 32.1, 32 x 32000 48.7 and 87.0)
  const bool one = cap <= kChooseLong || (cap <= kChooseOne && (int64_t)s.nseq * p.kv_heads >= 96);
  if (cap <= 4 * kChooseThreads)
    k_kv_choose<4><<<grid, kChooseThreads, 0, st>>>(p, s, budget, sinks, recent, src);
  else if (cap <= kChooseLong)
    k_kv_choose<16><<<grid, kChooseThreads, 0, st>>>(p, s, budget, sinks, recent, src);
  else if (one)
    k_kv_choose<32><<<grid, kChooseThreads, 0, st>>>(p, s, budget, sinks, recent, src);
  else {
    KvChooseLong l;
    l.segments = (cap + kSegment - 1) / kSegment;
    l.budget = budget, l.sinks = sinks, l.recent = recent;
    l.hist = c.choose_hist.as<uint32_t>();
    l.cut = c.choose_cut.as<KvCut>();
    l.counts = c.choose_counts.as<KvCounts>();
    l.list = c.choose_list.as<int32_t>();
    const dim3 g(l.segments, p.kv_heads, s.nseq);
    k_kv_choose_long<0><<<g, kChooseThreads, 0, st>>>(p, s, l, src);
    k_kv_choose_long<1><<<g, kChooseThreads, 0, st>>>(p, s, l, src);
    k_kv_choose_long<2><<<g, kChooseThreads, 0, st>>>(p, s, l, src);
    k_kv_choose_long<3><<<g, kChooseThreads, 0, st>>>(p, s, l, src);
    k_kv_choose_long<4><<<g, kChooseThreads, 0, st>>>(p, s, l, src);
    k_kv_fill<<<dim3((unsigned)blocks_of(budget), p.kv_heads, s.nseq), 256, 0, st>>>(
        budget, cap / 2, l.list, l.hist, src);
  }
  return hip_status(hipGetLastError(), "k_kv_choose");
}

Status launch_kv_compact(const KvPool& p, const KvSeqs& s, int budget, const int32_t* src,
                         hipStream_t st) {
  if (s.nseq == 0) return Status::ok();
  const dim3 grid((unsigned)blocks_of(budget), p.kv_heads, s.nseq);
  const int pieces = p.pitch * kv_elem_bytes(p.dtype) / 16;  // at most 64
  if (pieces <= 4) k_kv_compact<4><<<grid, 256, 0, st>>>(p, s, budget, src);
  else if (pieces <= 8) k_kv_compact<8><<<grid, 256, 0, st>>>(p, s, budget, src);
  else if (pieces <= 16) k_kv_compact<16><<<grid, 256, 0, st>>>(p, s, budget, src);
  else if (pieces <= 32) k_kv_compact<32><<<grid, 256, 0, st>>>(p, s, budget, src);
  else k_kv_compact<64><<<grid, 256, 0, st>>>(p, s, budget, src);
  return hip_status(hipGetLastError(), "k_kv_compact");
}

Status launch_kv_rope(float* q, float* k, int heads, int kv_heads, int hd, int q_stride,
                      int kv_stride, double theta, const KvPool& p, const KvSeqs& s, hipStream_t st) {
  if (s.nseq == 0 || hd < 2) return Status::ok();
  if (hd > kKvMaxHd) return Status::err(kUnsupported, "kv rope: head_dim above 256");
  k_kv_rope<<<s.nseq, 256, 0, st>>>(q, k, heads, kv_heads, hd, q_stride, kv_stride, theta, p, s);
  return hip_status(hipGetLastError(), "k_kv_rope");
}

Status launch_kv_advance(int nseq, int32_t* lens, int32_t* next_pos, const int32_t* counts, int add,
                         int cap, hipStream_t st) {
  if (nseq == 0) return Status::ok();
  k_kv_advance<<<(unsigned)blocks_of(nseq), 256, 0, st>>>(nseq, lens, next_pos, counts, add, cap);
  return hip_status(hipGetLastError(), "k_kv_advance");
}

}  // namespace wv
