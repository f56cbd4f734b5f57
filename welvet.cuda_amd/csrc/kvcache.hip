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

namespace wv {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float load_elem(const uint8_t* row, int dtype, int d) {
  if (dtype == kKvF32) return reinterpret_cast<const float*>(row)[d];
  if (dtype == kKvBF16) return float_of((uint32_t) reinterpret_cast<const uint16_t*>(row)[d] << 16);
  return decode_e4m3(row[d]);
}

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

__device__ __forceinline__ uint16_t bf16_bits(float f) {
  const uint32_t u = bits_of(f);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);  // NaN stays one
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);                  // nearest, ties to even
}

// Four elements of a row in the cache's type. Every lane of the group takes part
// (E4M3: in the row's maximum); those past the row (d >= pitch) store nothing.
__device__ __forceinline__ void store_row4(uint8_t* row, float* scale, v4f x, int dtype, int d,
                                           int pitch, int lanes) {
  if (dtype == kKvF32) {
    if (d < pitch) *reinterpret_cast<v4f*>(row + 4 * (size_t)d) = x;
  } else if (dtype == kKvBF16) {
    const uint32_t lo = bf16_bits(x[0]) | ((uint32_t)bf16_bits(x[1]) << 16);
    const uint32_t hi = bf16_bits(x[2]) | ((uint32_t)bf16_bits(x[3]) << 16);
    if (d < pitch) *reinterpret_cast<uint2*>(row + 2 * (size_t)d) = make_uint2(lo, hi);
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
    const float s = kv_e4m3_scale(float_of(m));
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w |= (uint32_t)canonical(kE4M3, encode_e4m3(x[j] / s)) << (8 * j);
    if (d < pitch) *reinterpret_cast<uint32_t*>(row + d) = w;
    if (d == 0) *scale = s;
  }
}

template <bool VEC>
__global__ __launch_bounds__(256) void k_kv_append(KvPool p, KvSeqs s, KvRows r, int lanes,
                                                   int64_t groups) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;
  const int d = 4 * (threadIdx.x & (lanes - 1));
  if (i >= groups) return;
  const int h = (int)(i % p.kv_heads);
  const int64_t t = i / p.kv_heads;  // token row
  const int b = (int)(t / r.rows), j = (int)(t % r.rows);
  if (r.counts && j >= r.counts[b]) return;
  const int cap = p.capacity();
  const int len = s.lens[b];
  const int e = kv_entries(len, 0, cap) + j;
  if (e >= cap) return;
  const int64_t row = kv_row(s.table + (size_t)b * p.max_pages, e, h, p.num_pages, p.kv_heads,
                             p.page_tokens);
  if (d == 0) {
    const size_t at = ((size_t)b * p.kv_heads + h) * cap + e;
    if (s.pos) s.pos[at] = (s.next_pos ? s.next_pos[b] : len < 0 ? 0 : len) + j;
    if (s.weight) s.weight[at] = 0.0f;
  }
  if (row < 0) return;
  const v4f kx = load_row4<VEC>(r.k + t * r.k_stride + (size_t)h * p.hd, d, p.hd);
  const v4f vx = load_row4<VEC>(r.v + t * r.v_stride + (size_t)h * p.hd, d, p.hd);
  const size_t at = (size_t)row * p.pitch * kv_elem_bytes(p.dtype);
  store_row4(p.k + at, p.ks + row, kx, p.dtype, d, p.pitch, lanes);
  store_row4(p.v + at, p.vs + row, vx, p.dtype, d, p.pitch, lanes);
}

// ---------------------------------------------------------------------------
// Read: entries first[b] + i as fp32, i < counts[b]; zero behind.
__global__ __launch_bounds__(256) void k_kv_read(KvPool p, KvSeqs s, int count,
                                                 const int32_t* __restrict__ first,
                                                 const int32_t* __restrict__ counts,
                                                 float* __restrict__ k, float* __restrict__ v,
                                                 int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int d = (int)(i % p.hd);
  const int64_t g = i / p.hd;
  const int h = (int)(g % p.kv_heads);
  const int64_t t = g / p.kv_heads;
  const int b = (int)(t / count), j = (int)(t % count);
  const int f = first ? first[b] : 0, c = counts ? counts[b] : count;
  float kx = 0.0f, vx = 0.0f;
  if (j < c && f >= 0 && f < p.capacity() - j) {
    const int64_t row = kv_row(s.table + (size_t)b * p.max_pages, f + j, h, p.num_pages, p.kv_heads,
                               p.page_tokens);
    if (row >= 0) {
      const size_t bytes = (size_t)p.pitch * kv_elem_bytes(p.dtype);
      kx = load_elem(p.k + (size_t)row * bytes, p.dtype, d);
      vx = load_elem(p.v + (size_t)row * bytes, p.dtype, d);
      if (p.dtype == kKvE4M3) kx *= p.ks[row], vx *= p.vs[row];
    }
  }
  k[i] = kx;
  v[i] = vx;
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
// only when a score exceeds it by more than 2^kSlack (weights of up to 2^8 lose
// nothing in fp32), so most tiles need no exchange between lanes.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));

constexpr float kSlack = 8.0f;

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
  int i = 0;
#pragma unroll
  for (; i + 4 <= N; i += 4) {
    const u32x4 x = *reinterpret_cast<const u32x4_a4*>(p + 4 * i);
#pragma unroll
    for (int k = 0; k < 4; ++k) w[i + k] = x[k];
  }
  if constexpr (N % 4 >= 2) {
    const auto x = *reinterpret_cast<const u32x2_a4*>(p + 4 * (N / 4 * 4));
    w[N / 4 * 4] = x[0], w[N / 4 * 4 + 1] = x[1];
  }
  if constexpr (N % 2 == 1) w[N - 1] = *reinterpret_cast<const uint32_t*>(p + 4 * (N - 1));
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

template <int DT, int HDP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HDP > 128 ? 1 : 2, 8)))
void k_kv_attend(KvPool p, KvSeqs s, KvAttend a, KvPart part) {
  using T = KvShape<DT, HDP>;
  constexpr int NSUB = T::NSUB, KT = 16 * NSUB, W = 4;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int group = p.heads / p.kv_heads, chunks = (group + 15) / 16;
  const int h = blockIdx.y / chunks, chunk = blockIdx.y % chunks, b = blockIdx.z;
  const int cols = group - 16 * chunk < 16 ? group - 16 * chunk : 16;
  const int head0 = h * group + 16 * chunk;
  const int cap = p.capacity();
  const int n = kv_entries(s.lens[b], a.tail, cap);
  const int qp = (s.next_pos ? s.next_pos[b] : n - a.tail) + a.tail - 1;
  const int32_t* table = s.table + (size_t)b * p.max_pages;
  const int32_t* pos = s.pos ? s.pos + ((size_t)b * p.kv_heads + h) * cap : nullptr;
  const KvRange range = kv_range(n, qp, pos == nullptr ? a.window : 0, KT, part.splits);
  const int t0 = range.first + (int)blockIdx.x * range.step;
  const int t1 = t0 + range.step < range.end ? t0 + range.step : range.end;
  if (blockIdx.x != 0 && t0 >= range.end) return;

  // queries: head c's values for this lane's part of the contraction
  const bool col_ok = c < cols;
  const float* qrow = a.q + (int64_t)b * a.q_stride + (int64_t)(head0 + (col_ok ? c : 0)) * p.hd;
  const float slope =
      a.alibi ? (float)(exp2(-8.0 * (double)(head0 + c + 1) / (double)p.heads) * kLog2e) : 0.0f;
  auto q_at = [&](int d) { return col_ok && d < p.hd ? qrow[d] : 0.0f; };
  float mult = a.scale2;
  float qf[DT == kKvF32 ? HDP / 4 : 1];
  bf16x8 qt[DT == kKvF32 ? 1 : T::KS][3];
  if constexpr (DT == kKvF32) {
#pragma unroll
    for (int i = 0; i < T::KL; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[4 * i + j] = q_at(16 * i + 4 * g + j);
  } else {
    float x[T::KS][8];
    float top = 0.0f;
#pragma unroll
    for (int ks = 0; ks < T::KS; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[ks][j] = q_at(DT == kKvBF16 ? 32 * ks + 8 * g + j : 64 * (ks / 2) + 16 * g + 8 * (ks % 2) + j);
        top = fmaxf(top, fabsf(x[ks][j]));
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // terms of values of about 1: the third one of a small query would fall
    // below bf16's normal range
    int e = (int)(bits_of(top) >> 23) - 127;
    e = e < -126 || e > 126 ? 0 : e;
    mult *= pow2f(e);
#pragma unroll
    for (int ks = 0; ks < T::KS; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        __bf16 t[3];
        split_bf16<3>(x[ks][j] * pow2f(-e), t);
#pragma unroll
        for (int k = 0; k < 3; ++k) qt[ks][k][j] = t[k];
      }
  }

  v4f acc[T::D];
#pragma unroll
  for (int d = 0; d < T::D; ++d) acc[d] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.0f;

  const int row_bytes = p.pitch * T::ELEM;
  const int koff = c * row_bytes + 16 * g;
  // (dims behind the row: any valid address; they are not written out)
  const int vcol = c * T::D * T::ELEM < row_bytes ? c * T::D * T::ELEM : 0;
  const int voff = 4 * g * row_bytes + vcol;

  // Pages of the tile's groups, stepping by the waves' tiles: index in the
  // table and entry in the page.
  const int step = W * KT, step_q = step / p.page_tokens, step_r = step - step_q * p.page_tokens;
  int pidx[NSUB], poff[NSUB];
#pragma unroll
  for (int u = 0; u < NSUB; ++u) {
    const int e = (t0 + wave) * KT + 16 * u;
    pidx[u] = e / p.page_tokens, poff[u] = e - pidx[u] * p.page_tokens;
  }
  // pool rows of a tile's groups; a group without entries or page: -1
  auto rows_of = [&](int t, int64_t (&row)[NSUB]) {
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      row[u] = -1;
      if (t < t1 && t * KT + 16 * u < n) {
        const int page = table[pidx[u]];
        if (page >= 0 && page < p.num_pages)
          row[u] = ((int64_t)page * p.kv_heads + h) * p.page_tokens + poff[u];
      }
      pidx[u] += step_q, poff[u] += step_r;
      if (poff[u] >= p.page_tokens) poff[u] -= p.page_tokens, ++pidx[u];
    }
  };
  u32x4 kr[NSUB][T::KL];
  auto load_k = [&](const int64_t (&row)[NSUB]) {
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      const uint8_t* base = p.k + (row[u] < 0 ? 0 : row[u]) * row_bytes;
#pragma unroll
      for (int i = 0; i < T::KL; ++i) {
        const bool in = i < T::KFULL || 64 * i + 16 * g < row_bytes;
        const u32x4 x = *reinterpret_cast<const u32x4*>(base + (in ? koff + 64 * i : 0));
        kr[u][i] = in ? x : u32x4{0, 0, 0, 0};
      }
    }
  };

  int64_t row[NSUB], next[NSUB];
  rows_of(t0 + wave, row);
  load_k(row);
  for (int t = t0 + wave; t < t1; t += W) {
    rows_of(t + W, next);
    uint32_t vr[4 * NSUB][T::VW];
    v4f ks[NSUB], vs[NSUB];
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      const int64_t r = row[u] < 0 ? 0 : row[u];
      const uint8_t* base = p.v + r * row_bytes;
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<T::VW>(vr[4 * u + i], base + voff + i * row_bytes);
      if constexpr (DT == kKvE4M3) {
        ks[u] = *reinterpret_cast<const v4f*>(p.ks + r + 4 * g);
        vs[u] = *reinterpret_cast<const v4f*>(p.vs + r + 4 * g);
      }
    }
    // scores, the small terms apart from the large one
    v4f x[NSUB];
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      v4f big = {0.f, 0.f, 0.f, 0.f}, small = {0.f, 0.f, 0.f, 0.f};
      if constexpr (DT == kKvF32) {
#pragma unroll
        for (int i = 0; i < T::KL; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v4f& to = i & 1 ? small : big;
            to = __builtin_amdgcn_mfma_f32_16x16x4f32(float_of(kr[u][i][j]), qf[4 * i + j], to, 0, 0, 0);
          }
      } else {
#pragma unroll
        for (int ks_ = 0; ks_ < T::KS; ++ks_) {
          bf16x8 k8;
          if constexpr (DT == kKvBF16) {
            k8 = __builtin_bit_cast(bf16x8, kr[u][ks_]);
          } else {
            const uint32_t w0 = kr[u][ks_ / 2][2 * (ks_ % 2)], w1 = kr[u][ks_ / 2][2 * (ks_ % 2) + 1];
            k8 = __builtin_bit_cast(bf16x8, u32x4{cvt_e4m3<false>(w0), cvt_e4m3<true>(w0),
                                                  cvt_e4m3<false>(w1), cvt_e4m3<true>(w1)});
          }
          small = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8, qt[ks_][2], small, 0, 0, 0);
          big = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8, qt[ks_][0], big, 0, 0, 0);
          small = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8, qt[ks_][1], small, 0, 0, 0);
        }
      }
      x[u] = (big + small) * mult;
      if constexpr (DT == kKvE4M3) x[u] *= ks[u];
    }
    const bool rows_ok = row[0] >= 0 && row[NSUB - 1] >= 0;
    const bool whole = rows_ok && (t + 1) * KT <= n && a.window <= 0;
    if (a.alibi || a.window > 0) {
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
    if (!whole) {
      // entries that are not seen: weight 0, and no NaN of theirs times it
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = t * KT + 16 * u + 4 * g + i;
          bool seen = row[u] >= 0 && e < n;
          if (a.window > 0) seen = seen && qp - (pos ? pos[e < cap ? e : 0] : e) < a.window;
          if (!seen) {
            x[u][i] = -INFINITY;
#pragma unroll
            for (int w = 0; w < T::VW; ++w) vr[4 * u + i][w] = 0;
            if constexpr (DT == kKvE4M3) vs[u][i] = 0.0f;
          }
        }
    }
    if (part.scores && col_ok) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        const int e = t * KT + 16 * u + 4 * g;
        if (e < cap)  // (a capacity is whole groups of 16)
          *reinterpret_cast<v4f*>(part.scores + ((size_t)b * p.heads + head0 + c) * cap + e) = x[u];
      }
    }
    if (t + W < t1) load_k(next);

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
        if constexpr (DT == kKvE4M3) w[4 * u + i] *= vs[u][i];
      }
    if constexpr (DT == kKvF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < T::D; ++d)
          acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(float_of(vr[i][d]), w[i], acc[d], 0, 0, 0);
    } else {
      bf16x8 pt[3];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        __bf16 t3[3];
        split_bf16<3>(w[j], t3);
#pragma unroll
        for (int k = 0; k < 3; ++k) pt[k][j] = t3[k];
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
#pragma unroll
    for (int u = 0; u < NSUB; ++u) row[u] = next[u];
  }

  // The waves' sums meet: waves 2 and 3 hand theirs to 0 and 1, then 1 to 0.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  constexpr int STRIDE = HDP + 4;
  __shared__ float ml[W][16][2];
  __shared__ __attribute__((aligned(16))) float sums[2][16][STRIDE];
  if (g == 0) ml[wave][c][0] = m, ml[wave][c][1] = l;
  __syncthreads();
  float M = -INFINITY, L = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) M = fmaxf(M, ml[w][c][0]);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float mw = ml[w][c][0];
    L += ml[w][c][1] * (mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - M));
  }
  const float mine = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - M);
#pragma unroll
  for (int d = 0; d < T::D; ++d) acc[d] *= mine;
#pragma unroll
  for (int half = 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half && col_ok) {
#pragma unroll
      for (int d = 0; d < T::D; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[wave - half][c][(4 * g + i) * T::D + d] = acc[d][i];
    }
    __syncthreads();
    if (wave < half && col_ok) {
#pragma unroll
      for (int d = 0; d < T::D; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[d][i] += sums[wave][c][(4 * g + i) * T::D + d];
    }
    __syncthreads();
  }
  if (wave != 0 || !col_ok) return;
  const size_t hi = (size_t)b * p.heads + head0 + c;
  float* to;
  float f = 1.0f;
  if (range.parts <= 1) {
    to = a.out + (int64_t)b * a.out_stride + (int64_t)(head0 + c) * p.hd;
    f = L == 0.0f ? 0.0f : 1.0f / L;
    if (g == 0) {
      const float lse2 = L == 0.0f ? -INFINITY : M + __builtin_amdgcn_logf(L);
      if (a.lse) a.lse[hi] = lse2 * kLn2;
      if (part.lse2) part.lse2[hi] = lse2;
    }
  } else {
    const size_t at = hi * part.splits + blockIdx.x;
    to = part.out + at * p.hd;
    if (g == 0) part.ml[2 * at] = M, part.ml[2 * at + 1] = L;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int d = 0; d < T::D; ++d) {
      const int dim = (4 * g + i) * T::D + d;
      if (dim < p.hd) to[dim] = acc[d][i] * f;
    }
}

// Joins the parts of one (sequence, head).
__global__ __launch_bounds__(256) void k_kv_join(KvPool p, KvSeqs s, KvAttend a, KvPart part, int kt) {
  const int j = blockIdx.x, b = blockIdx.y, h = j / (p.heads / p.kv_heads);
  const int n = kv_entries(s.lens[b], a.tail, p.capacity());
  const int qp = (s.next_pos ? s.next_pos[b] : n - a.tail) + a.tail - 1;
  const KvRange range = kv_range(n, qp, s.pos == nullptr ? a.window : 0, kt, part.splits);
  if (range.parts <= 1) return;
  (void)h;
  const size_t hi = (size_t)b * p.heads + j, at = hi * part.splits;
  float M = -INFINITY, L = 0.0f;
  for (int i = 0; i < range.parts; ++i) M = fmaxf(M, part.ml[2 * (at + i)]);
  for (int i = 0; i < range.parts; ++i) {
    const float mi = part.ml[2 * (at + i)];
    L += part.ml[2 * (at + i) + 1] * (mi == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mi - M));
  }
  for (int d = threadIdx.x; d < p.hd; d += 256) {
    float o = 0.0f;
    for (int i = 0; i < range.parts; ++i) {
      const float mi = part.ml[2 * (at + i)];
      o += part.out[(at + i) * p.hd + d] * (mi == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mi - M));
    }
    a.out[(int64_t)b * a.out_stride + (int64_t)j * p.hd + d] = L == 0.0f ? 0.0f : o / L;
  }
  if (threadIdx.x == 0) {
    const float lse2 = L == 0.0f ? -INFINITY : M + __builtin_amdgcn_logf(L);
    if (a.lse) a.lse[hi] = lse2 * kLn2;
    if (part.lse2) part.lse2[hi] = lse2;
  }
}

// Running sums: weight[e] += the weights of the K/V head's query heads, from
// the scores and the sums of e^score.
__global__ __launch_bounds__(256) void k_kv_track(KvPool p, KvSeqs s, KvAttend a, KvPart part, int kt) {
  const int h = blockIdx.y, b = blockIdx.z, cap = p.capacity(), group = p.heads / p.kv_heads;
  const int n = kv_entries(s.lens[b], a.tail, cap);
  const int qp = (s.next_pos ? s.next_pos[b] : n - a.tail) + a.tail - 1;
  const KvRange range = kv_range(n, qp, s.pos == nullptr ? a.window : 0, kt, part.splits);
  const float* lse2 = part.lse2 + (size_t)b * p.heads + (size_t)h * group;
  const float* sc = part.scores + ((size_t)b * p.heads + (size_t)h * group) * cap;
  for (int e = range.first * kt + blockIdx.x * 256 + threadIdx.x; e < n; e += gridDim.x * 256) {
    float w = 0.0f;
    for (int j = 0; j < group; ++j) {
      const float x = sc[(size_t)j * cap + e];
      w += x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - lse2[j]);
    }
    s.weight[((size_t)b * p.kv_heads + h) * cap + e] += w;
  }
}

// ---------------------------------------------------------------------------
// Choice of the entries to keep: the key of the `budget`-th entry bit by bit,
// then the kept entries from behind the budget into the holes below it, both
// in index order. One workgroup per (sequence, K/V head).
constexpr int kChooseThreads = 1024;

__device__ __forceinline__ int block_count(bool x, int* red) {
  const unsigned long long bits = __ballot(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __popcll(bits);
  __syncthreads();
  int n = 0;
  for (int w = 0; w < kChooseThreads / 64; ++w) n += red[w];
  return n;
}

// Flags before this thread's in the workgroup; total: all of them.
__device__ __forceinline__ int block_rank(bool x, int* red, int& total) {
  const unsigned long long bits = __ballot(x);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) red[wave] = __popcll(bits);
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < kChooseThreads / 64; ++w) {
    if (w == wave) before = total;
    total += red[w];
  }
  return before + __popcll(bits & ((1ull << lane) - 1));
}

__global__ __launch_bounds__(kChooseThreads) void k_kv_choose(KvPool p, KvSeqs s, int budget,
                                                              int sinks, int recent,
                                                              int32_t* __restrict__ out) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, cap = p.capacity();
  __shared__ int red[kChooseThreads / 64];
  const int n = kv_entries(s.lens[b], 0, cap);
  const int end = s.next_pos ? s.next_pos[b] : n;
  const size_t base = ((size_t)b * p.kv_heads + h) * cap;
  const float* weight = s.weight + base;
  const int32_t* pos = s.pos ? s.pos + base : nullptr;
  int32_t* src = out + ((size_t)b * p.kv_heads + h) * budget;
  if (n <= budget) {
    for (int j = tid; j < budget; j += kChooseThreads) src[j] = j < n ? j : -1;
    return;
  }
  auto key = [&](int e) {
    const int q = pos ? pos[e] : e;
    if (q < sinks || (int64_t)q >= (int64_t)end - recent) return kKvKeyFirst;
    return kv_weight_key(weight[e]);
  };
  uint32_t least = 0;  // the largest key that `budget` entries reach
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = least | (1u << bit);
    int c = 0;
    for (int e0 = 0; e0 < n; e0 += kChooseThreads)
      c += block_count(e0 + tid < n && key(e0 + tid) >= t, red);
    if (c >= budget) least = t;
  }
  int above = 0;
  for (int e0 = 0; e0 < n; e0 += kChooseThreads)
    above += block_count(e0 + tid < n && key(e0 + tid) > least, red);
  const int ties = budget - above;  // of the entries at `least`, the first ones
  int equal = 0;  // entries at `least` below the budget
  for (int e0 = 0; e0 < budget; e0 += kChooseThreads)
    equal += block_count(e0 + tid < budget && key(e0 + tid) == least, red);
  // the kept entries from behind the budget, in order, listed in src from its
  // start (there are as many holes below the budget: the list fits)
  int holes = 0, seen = equal;
  for (int e0 = budget; e0 < n; e0 += kChooseThreads) {
    const int e = e0 + tid;
    const uint32_t k = e < n ? key(e) : 0;
    int total;
    const int r = block_rank(e < n && k == least, red, total);
    const bool kept = e < n && (k > least || (k == least && seen + r < ties));
    seen += total;
    const int at = block_rank(kept, red, total);
    if (kept) src[holes + at] = e;
    holes += total;
  }
  // The slots from the last to the first: the hole of rank i takes src[i],
  // and i is at most its own index, so what a run of slots overwrites is
  // listed for its own holes (read before) or for those already done.
  seen = equal;
  int left = holes;
  for (int e0 = (budget - 1) / kChooseThreads * kChooseThreads; e0 >= 0; e0 -= kChooseThreads) {
    const int e = e0 + tid;
    const bool in = e < budget;
    const uint32_t k = in ? key(e) : 0;
    int total;
    const int r = block_rank(in && k == least, red, total);
    seen -= total;
    const bool hole = in && !(k > least || (k == least && seen + r < ties));
    const int at = block_rank(hole, red, total);
    left -= total;
    const int from = hole ? src[left + at] : e;
    __syncthreads();
    if (in) src[e] = from;
  }
}

// ---------------------------------------------------------------------------
// Compaction: one wave per (sequence, K/V head, slot).
__global__ __launch_bounds__(256) void k_kv_compact(KvPool p, KvSeqs s, int budget,
                                                    const int32_t* __restrict__ src, int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 6;
  const int lane = threadIdx.x & 63;
  if (i >= n) return;
  const int j = (int)(i % budget);
  const int64_t bh = i / budget;
  const int h = (int)(bh % p.kv_heads), b = (int)(bh / p.kv_heads);
  const int e = src[i], cap = p.capacity();
  if (e < budget || e >= cap || j >= cap) return;  // its own, none, or outside
  const int32_t* table = s.table + (size_t)b * p.max_pages;
  const int64_t from = kv_row(table, e, h, p.num_pages, p.kv_heads, p.page_tokens);
  const int64_t to = kv_row(table, j, h, p.num_pages, p.kv_heads, p.page_tokens);
  if (lane == 0) {
    const size_t base = (size_t)bh * cap;
    if (s.weight) s.weight[base + j] = s.weight[base + e];
    if (s.pos) s.pos[base + j] = s.pos[base + e];
  }
  if (from < 0 || to < 0) return;
  const int bytes = p.pitch * kv_elem_bytes(p.dtype);
  for (int o = 16 * lane; o < bytes; o += 16 * 64) {
    *reinterpret_cast<v4f*>(p.k + (size_t)to * bytes + o) =
        *reinterpret_cast<const v4f*>(p.k + (size_t)from * bytes + o);
    *reinterpret_cast<v4f*>(p.v + (size_t)to * bytes + o) =
        *reinterpret_cast<const v4f*>(p.v + (size_t)from * bytes + o);
  }
  if (p.dtype == kKvE4M3 && lane == 0) {
    p.ks[to] = p.ks[from];
    p.vs[to] = p.vs[from];
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
  // every call's parts fit: splits * nseq * kv_heads * chunks stays below the
  // workgroups that the rule aims at wherever there is more than one part
  const size_t parts = (size_t)kKvWorkgroups * 16;
  WV_TRY(c->part.alloc(parts * hd * sizeof(float)));
  WV_TRY(c->part_ml.alloc(parts * 2 * sizeof(float)));
  WV_HIP(hipStreamSynchronize(st));
  p.k = c->k.as<uint8_t>(), p.v = c->v.as<uint8_t>();
  p.ks = c->ks.as<float>(), p.vs = c->vs.as<float>();
  return Status::ok();
}

Status launch_kv_append(const KvPool& p, const KvSeqs& s, const KvRows& r, hipStream_t st) {
  if (s.nseq == 0 || r.rows == 0) return Status::ok();
  int lanes = 1;
  while (4 * lanes < p.pitch) lanes *= 2;
  const int64_t groups = (int64_t)s.nseq * r.rows * p.kv_heads;
  const int64_t blocks = blocks_of(groups * lanes);
  if (blocks > INT32_MAX) return Status::err(kInvalid, "kv append: too many rows in one call");
  const bool vec = p.hd % 4 == 0 && r.k_stride % 4 == 0 && r.v_stride % 4 == 0 &&
                   ((uintptr_t)r.k | (uintptr_t)r.v) % 16 == 0;
  if (vec)
    k_kv_append<true><<<(unsigned)blocks, 256, 0, st>>>(p, s, r, lanes, groups);
  else
    k_kv_append<false><<<(unsigned)blocks, 256, 0, st>>>(p, s, r, lanes, groups);
  return hip_status(hipGetLastError(), "k_kv_append");
}

Status launch_kv_read(const KvPool& p, const KvSeqs& s, int count, const int32_t* first,
                      const int32_t* counts, float* k, float* v, hipStream_t st) {
  const int64_t n = (int64_t)s.nseq * count * p.kv_heads * p.hd;
  if (n == 0) return Status::ok();
  if (blocks_of(n) > INT32_MAX) return Status::err(kInvalid, "kv read: too many entries in one call");
  k_kv_read<<<(unsigned)blocks_of(n), 256, 0, st>>>(p, s, count, first, counts, k, v, n);
  return hip_status(hipGetLastError(), "k_kv_read");
}

template <int DT>
Status launch_attend(int hd, dim3 grid, const KvPool& p, const KvSeqs& s, const KvAttend& a,
                     const KvPart& part, hipStream_t st) {
#define WV_KV_HD(N) k_kv_attend<DT, N><<<grid, 256, 0, st>>>(p, s, a, part)
  if constexpr (DT == kKvE4M3) {
    if (hd <= 64) WV_KV_HD(64);
    else if (hd <= 128) WV_KV_HD(128);
    else if (hd <= 192) WV_KV_HD(192);
    else WV_KV_HD(256);
  } else {
    if (hd <= 32) WV_KV_HD(32);
    else if (hd <= 64) WV_KV_HD(64);
    else if (hd <= 96) WV_KV_HD(96);
    else if (hd <= 128) WV_KV_HD(128);
    else if (hd <= 192) WV_KV_HD(192);
    else WV_KV_HD(256);
  }
#undef WV_KV_HD
  return hip_status(hipGetLastError(), "k_kv_attend");
}

Status kv_attend(const KvCache& c, const KvSeqs& s, const KvAttend& a, hipStream_t st) {
  if (s.nseq == 0) return Status::ok();
  const KvPool& p = c.pool;
  const int kt = p.dtype == kKvF32 ? 16 : 32;
  KvPart part;
  part.splits = kv_splits(s.nseq, p.kv_heads, p.heads / p.kv_heads, p.capacity());
  part.out = c.part.as<float>();
  part.ml = c.part_ml.as<float>();
  if (s.weight) {
    part.scores = c.scores.as<float>();
    part.lse2 = c.lse2.as<float>();
  }
  const dim3 grid(part.splits, p.kv_heads * kv_chunks(p.heads / p.kv_heads), s.nseq);
  WV_TRY(p.dtype == kKvF32    ? launch_attend<kKvF32>(p.hd, grid, p, s, a, part, st)
         : p.dtype == kKvBF16 ? launch_attend<kKvBF16>(p.hd, grid, p, s, a, part, st)
                              : launch_attend<kKvE4M3>(p.hd, grid, p, s, a, part, st));
  if (part.splits > 1) {
    k_kv_join<<<dim3(p.heads, s.nseq), 256, 0, st>>>(p, s, a, part, kt);
    WV_TRY(hip_status(hipGetLastError(), "k_kv_join"));
  }
  if (!s.weight) return Status::ok();
  const int blocks = (p.capacity() + 255) / 256;
  k_kv_track<<<dim3(blocks < 64 ? blocks : 64, p.kv_heads, s.nseq), 256, 0, st>>>(p, s, a, part, kt);
  return hip_status(hipGetLastError(), "k_kv_track");
}

Status launch_kv_choose(const KvPool& p, const KvSeqs& s, int budget, int sinks, int recent,
                        int32_t* src, hipStream_t st) {
  if (s.nseq == 0) return Status::ok();
  k_kv_choose<<<dim3(p.kv_heads, s.nseq), kChooseThreads, 0, st>>>(p, s, budget, sinks, recent, src);
  return hip_status(hipGetLastError(), "k_kv_choose");
}

Status launch_kv_compact(const KvPool& p, const KvSeqs& s, int budget, const int32_t* src,
                         hipStream_t st) {
  const int64_t n = (int64_t)s.nseq * p.kv_heads * budget;
  if (n == 0) return Status::ok();
  if (blocks_of(n * 64) > INT32_MAX) return Status::err(kInvalid, "kv compact: too many slots in one call");
  k_kv_compact<<<(unsigned)blocks_of(n * 64), 256, 0, st>>>(p, s, budget, src, n);
  return hip_status(hipGetLastError(), "k_kv_compact");
}

Status launch_kv_advance(int nseq, int32_t* lens, int32_t* next_pos, const int32_t* counts, int add,
                         int cap, hipStream_t st) {
  if (nseq == 0) return Status::ok();
  k_kv_advance<<<(unsigned)blocks_of(nseq), 256, 0, st>>>(nseq, lens, next_pos, counts, add, cap);
  return hip_status(hipGetLastError(), "k_kv_advance");
}

}  // namespace wv
