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

namespace wv {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

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
// Attention, one workgroup per (sequence, query head): scores of all entries
// into scratch, their maximum and sum, then the values.
// The larger; NaN where one is.
__device__ __forceinline__ float max_nan(float a, float b) { return b > a || b != b ? b : a; }

__device__ __forceinline__ float block_max(float x, float* red) {
  for (int off = 32; off > 0; off >>= 1) x = max_nan(x, __shfl_xor(x, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return max_nan(max_nan(red[0], red[1]), max_nan(red[2], red[3]));
}

__device__ __forceinline__ float block_sum(float x, float* red) {
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void k_kv_attend(KvPool p, KvSeqs s, KvAttend a, float* scores) {
  const int j = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int group = p.heads / p.kv_heads, h = j / group, cap = p.capacity();
  __shared__ float qs[kKvMaxHd];
  __shared__ float red[4];
  for (int d = tid; d < p.hd; d += 256) qs[d] = a.q[b * a.q_stride + (size_t)j * p.hd + d];
  __syncthreads();
  const int n = kv_entries(s.lens[b], a.tail, cap);
  const int qp = (s.next_pos ? s.next_pos[b] : n - a.tail) + a.tail - 1;
  const int32_t* table = s.table + (size_t)b * p.max_pages;
  const int32_t* pos = s.pos ? s.pos + ((size_t)b * p.kv_heads + h) * cap : nullptr;
  float* sc = scores + ((size_t)b * p.heads + j) * cap;
  const size_t bytes = (size_t)p.pitch * kv_elem_bytes(p.dtype);
  const float slope = a.alibi ? (float)exp2(-8.0 * (j + 1) / p.heads) : 0.0f;
  float m = -INFINITY;
  for (int e = tid; e < n; e += 256) {
    const int64_t row = kv_row(table, e, h, p.num_pages, p.kv_heads, p.page_tokens);
    const int ahead = qp - (pos ? pos[e] : e);
    float x = -INFINITY;
    if (row >= 0 && (a.window <= 0 || ahead < a.window)) {
      x = 0.0f;
      for (int d = 0; d < p.hd; ++d)
        x = fmaf(qs[d], load_elem(p.k + (size_t)row * bytes, p.dtype, d), x);
      if (p.dtype == kKvE4M3) x *= p.ks[row];
      x = x * a.scale - slope * fabsf((float)ahead);
    }
    sc[e] = x;
    m = max_nan(m, x);
  }
  m = block_max(m, red);
  float l = 0.0f;
  for (int e = tid; e < n; e += 256) {
    const float w = sc[e] == -INFINITY ? 0.0f : expf(sc[e] - m);
    sc[e] = w;
    l += w;
  }
  l = block_sum(l, red);
  const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  for (int e = tid; e < n; e += 256) sc[e] = sc[e] == 0.0f ? 0.0f : sc[e] * inv;
  __syncthreads();
  for (int d = tid; d < p.hd; d += 256) {
    // eight sums, so that the rounding errors of long ones stay small
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int e0 = 0; e0 < n; e0 += 8)
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int e = e0 + u;
        const float w = e < n ? sc[e] : 0.0f;
        if (w == 0.0f) continue;
        const int64_t row = kv_row(table, e, h, p.num_pages, p.kv_heads, p.page_tokens);
        if (row < 0) continue;
        float x = load_elem(p.v + (size_t)row * bytes, p.dtype, d);
        if (p.dtype == kKvE4M3) x *= p.vs[row];
        o[u] = fmaf(w, x, o[u]);
      }
    a.out[b * a.out_stride + (size_t)j * p.hd + d] =
        ((o[0] + o[1]) + (o[2] + o[3])) + ((o[4] + o[5]) + (o[6] + o[7]));
  }
  if (a.lse && tid == 0) a.lse[(size_t)b * p.heads + j] = l == 0.0f ? -INFINITY : m + logf(l);
}

// Running sums: weight[e] += the weights of the K/V head's query heads.
__global__ __launch_bounds__(256) void k_kv_track(KvPool p, KvSeqs s, int tail, const float* scores) {
  const int h = blockIdx.y, b = blockIdx.z, cap = p.capacity(), group = p.heads / p.kv_heads;
  const int n = kv_entries(s.lens[b], tail, cap);
  for (int e = blockIdx.x * 256 + threadIdx.x; e < n; e += gridDim.x * 256) {
    float w = 0.0f;
    for (int g = 0; g < group; ++g)
      w += scores[((size_t)b * p.heads + (size_t)h * group + g) * cap + e];
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
    WV_TRY(b->alloc(bytes));
    WV_HIP(hipMemsetAsync(b->p, 0, bytes, st));
  }
  if (dtype == kKvE4M3)
    for (DevBuf* b : {&c->ks, &c->vs}) {
      WV_TRY(b->alloc(rows * sizeof(float)));
      WV_HIP(hipMemsetAsync(b->p, 0, rows * sizeof(float), st));
    }
  WV_TRY(c->scores.alloc((size_t)max_seqs * heads * p.capacity() * sizeof(float)));
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

Status kv_attend(const KvCache& c, const KvSeqs& s, const KvAttend& a, hipStream_t st) {
  if (s.nseq == 0) return Status::ok();
  const KvPool& p = c.pool;
  float* scores = c.scores.as<float>();
  k_kv_attend<<<dim3(p.heads, s.nseq), 256, 0, st>>>(p, s, a, scores);
  WV_TRY(hip_status(hipGetLastError(), "k_kv_attend"));
  if (!s.weight) return Status::ok();
  const int blocks = (p.capacity() + 255) / 256;
  k_kv_track<<<dim3(blocks < 64 ? blocks : 64, p.kv_heads, s.nseq), 256, 0, st>>>(p, s, a.tail, scores);
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
