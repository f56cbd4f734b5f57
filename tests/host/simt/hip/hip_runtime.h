// A stand-in for the HIP runtime on the CPU: device memory is host memory
// between guard pages, and a kernel runs lane by lane on stacks of its own that
// meet at cross-lane operations and barriers. For kernels of one-dimensional
// workgroups whose waves reach those operations with all their live lanes.
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#define __host__
#define __device__
#define __global__ __attribute__((noinline))
#define __shared__ static  // workgroups run one after the other
#define __launch_bounds__(x)
#define __forceinline__ inline
#define amdgpu_waves_per_eu(low, high) unused

struct dim3 {
  unsigned x, y, z;
  dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};
struct uint2 {
  uint32_t x, y;
};
inline uint2 make_uint2(uint32_t x, uint32_t y) { return uint2{x, y}; }

typedef int hipError_t;
typedef void* hipStream_t;
enum { hipSuccess = 0 };
extern "C" void* simt_alloc(size_t bytes);
extern "C" void simt_free(void* p);
template <class T>
int hipMalloc(T** p, size_t n) {
  *p = static_cast<T*>(simt_alloc(n));
  return *p ? 0 : 2;
}
inline int hipFree(void* p) { return simt_free(p), 0; }
inline int hipMemsetAsync(void* p, int v, size_t n, hipStream_t) { return memset(p, v, n), 0; }
inline int hipStreamSynchronize(hipStream_t) { return 0; }
inline int hipGetLastError() { return 0; }
inline const char* hipGetErrorString(int) { return "error"; }

namespace simt {

enum Stop { kRuns, kWaveOp, kBarrier };
struct Lane {
  void* sp;
  char* stack;
  bool done;
  Stop stop;
  int line;      // of the operation it waits at
  unsigned ops;  // cross-lane operations so far
  dim3 tid;
  int id;
};
// What the lanes of a wave hand in at an operation; two in turn, as lanes read
// one operation's while others are at the next.
struct Wave {
  unsigned char given[2][64][32];
  bool live[2][64];
};
extern Lane* cur;
extern dim3 block_idx, block_dim, grid_dim;
extern Wave waves[16];
// Called before every launch (0) and every workgroup (1), null: not at all.
extern void (*hook)(int kind);
[[noreturn]] void fail(const char* what);
void run_block(void (*fn)(void*), void* arg, int threads);
void wave_op(int line);
void barrier(int line);

inline int lane() { return cur->id & 63; }
template <class T>
int give(const T& v, int at = 0) {
  static_assert(sizeof(T) <= 32, "");
  Wave& w = waves[cur->id >> 6];
  const int g = cur->ops & 1;
  memcpy(w.given[g][lane()] + at, &v, sizeof v);
  w.live[g][lane()] = true;
  return g;
}
template <class T>
bool take(int g, int from, T* v, int at = 0) {
  const Wave& w = waves[cur->id >> 6];
  memset(v, 0, sizeof *v);
  if (from < 0 || from > 63 || !w.live[g][from]) return false;
  memcpy(v, w.given[g][from] + at, sizeof *v);
  return true;
}
template <class T>
T from_lane(T v, int from, int line) {
  const int g = give(v);
  wave_op(line);
  T r;
  take(g, from, &r);
  return r;
}
inline unsigned long long ballot(bool b, int line) {
  const int g = give((int)b);
  wave_op(line);
  unsigned long long m = 0;
  for (int i = 0, x; i < 64; ++i)
    if (take(g, i, &x) && x) m |= 1ull << i;
  return m;
}
inline int readlane(int v, int from, int line) {
  const int g = give(v);
  give(from, 8);
  wave_op(line);
  int r;
  for (int i = 0, other; i < 64; ++i)
    if (take(g, i, &other, 8) && other != from) fail("readlane of differing lanes");
  if (!take(g, from, &r)) fail("readlane of no live lane");
  return r;
}
inline int readfirstlane(int v, int line) {
  const int g = give(v);
  wave_op(line);
  for (int i = 0, r; i < 64; ++i)
    if (take(g, i, &r)) return r;
  return v;
}
inline int dpp(int old, int v, int ctrl, int rows, int line) {
  const int g = give(v);
  wave_op(line);
  const int l = lane(), row = l / 16, in = l % 16, n = ctrl & 15;
  if (!(rows >> row & 1)) return old;
  int from = -1;
  if (ctrl < 0x100) from = (l & ~3) | (ctrl >> (2 * (l & 3)) & 3);           // quad_perm
  else if (ctrl > 0x100 && ctrl < 0x110) from = in + n < 16 ? l + n : -1;    // row_shl
  else if (ctrl > 0x110 && ctrl < 0x120) from = in >= n ? l - n : -1;        // row_shr
  else if (ctrl > 0x120 && ctrl < 0x130) from = 16 * row + ((in - n) & 15);  // row_ror
  else if (ctrl == 0x142) from = 16 * row - 1;                               // row_bcast:15
  else if (ctrl == 0x143) from = row >= 2 ? 31 : -1;                         // row_bcast:31
  else fail("DPP control");
  int r;
  return take(g, from, &r) ? r : old;
}
inline int ds_permute(int address, int v, int line) {
  const int g = give(v);
  give(address, 8);
  wave_op(line);
  int r = 0;
  for (int i = 0, to; i < 64; ++i)
    if (take(g, i, &to, 8) && (to / 4 & 63) == lane()) take(g, i, &r);
  return r;
}
inline uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  const uint64_t both = (uint64_t)hi << 32 | lo;
  uint32_t r = 0;
  for (int i = 0; i < 4; ++i) {
    const unsigned s = sel >> (8 * i) & 255;
    if (s > 7) fail("byte selector");
    r |= (uint32_t)(both >> (8 * s) & 255) << (8 * i);
  }
  return r;
}

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
inline float e4m3(unsigned c) {
  const int e = c >> 3 & 15, m = c & 7;
  const float a = e == 15 && m == 7 ? NAN : e ? ldexpf(1.0f + m / 8.0f, e - 7) : ldexpf(m / 8.0f, -6);
  return c & 128 ? -a : a;
}
inline v2f cvt_f32_fp8(uint32_t w, bool hi) {
  w >>= hi ? 16 : 0;
  return v2f{e4m3(w & 255), e4m3(w >> 8 & 255)};
}
inline v2b cvt_bf16_fp8(uint32_t w, float s, bool hi) {
  const v2f x = cvt_f32_fp8(w, hi);
  return v2b{(__bf16)(x[0] * s), (__bf16)(x[1] * s)};
}
// D = A B + C of 16 x 16: lane 16 q + r holds row r of A and column r of B, K
// elements N q .. N q + N - 1, and rows 4 q + i of column r of C.
template <int N, class T>
v4f mfma(const T& a, const T& b, v4f c, int line) {
  const int g = give(a);
  give(b, 16);
  wave_op(line);
  const auto& given = waves[cur->id >> 6].given[g];
  const int r = lane() % 16, row = lane() / 16 * 4;
  for (int q = 0; q < 4; ++q) {
    T x, y;
    memcpy(&y, given[16 * q + r] + 16, sizeof y);
    for (int i = 0; i < 4; ++i) {
      memcpy(&x, given[16 * q + row + i], sizeof x);
      if constexpr (N == 1) {
        c[i] += x * y;
      } else {
        typedef float vf __attribute__((ext_vector_type(N)));
        const vf p = __builtin_convertvector(x, vf) * __builtin_convertvector(y, vf);
        for (int k = 0; k < N; ++k) c[i] += p[k];
      }
    }
  }
  return c;
}

template <class F>
struct Launch {
  F fn;
  dim3 grid, block;
  template <class... A>
  void operator()(A... args) {
    if (block.x > 1024 || block.y != 1 || block.z != 1 || !grid.x || !grid.y || !grid.z ||
        grid.y > 65535 || grid.z > 65535)
      fail("shape of a launch");
    if (hook) hook(0);
    grid_dim = grid, block_dim = block;
    auto call = [&] { fn(args...); };
    using C = decltype(call);
    for (unsigned z = 0; z < grid.z; ++z)
      for (unsigned y = 0; y < grid.y; ++y)
        for (unsigned x = 0; x < grid.x; ++x) {
          if (hook) hook(1);
          block_idx = dim3(x, y, z);
          run_block([](void* p) { (*static_cast<C*>(p))(); }, &call, (int)block.x);
        }
  }
};
template <class F>
Launch<F> launch(F fn, dim3 grid, dim3 block, size_t, hipStream_t) {
  return Launch<F>{fn, grid, block};
}

}  // namespace simt

inline uint32_t atomicAdd(uint32_t* p, uint32_t v) {
  const uint32_t old = *p;
  *p += v;
  return old;
}

#define threadIdx (simt::cur->tid)
#define blockIdx simt::block_idx
#define blockDim simt::block_dim
#define gridDim simt::grid_dim
#define __syncthreads() simt::barrier(__LINE__)
#define __shfl_xor(v, off, width) simt::from_lane(v, simt::lane() ^ (off), __LINE__)
#define __shfl(v, from, width) simt::from_lane(v, from, __LINE__)
#define __ballot(b) simt::ballot(b, __LINE__)
#define __popcll(x) __builtin_popcountll(x)
#define __float_as_int(f) __builtin_bit_cast(int, f)
#define __int_as_float(i) __builtin_bit_cast(float, i)
#define __builtin_amdgcn_readlane(v, from) simt::readlane(v, from, __LINE__)
#define __builtin_amdgcn_readfirstlane(v) simt::readfirstlane(v, __LINE__)
#define __builtin_amdgcn_update_dpp(old, v, ctrl, rows, banks, bound) simt::dpp(old, v, ctrl, rows, __LINE__)
#define __builtin_amdgcn_mov_dpp(v, ctrl, rows, banks, bound) simt::dpp(0, v, ctrl, rows, __LINE__)
#define __builtin_amdgcn_ds_permute(address, v) simt::ds_permute(address, v, __LINE__)
#define __builtin_amdgcn_perm(hi, lo, sel) simt::perm(hi, lo, sel)
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_logf(x) log2f(x)
#define __builtin_amdgcn_cvt_pk_f32_fp8(w, hi) simt::cvt_f32_fp8(w, hi)
#define __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, hi) simt::cvt_bf16_fp8(w, s, hi)
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) simt::mfma<8>(a, b, c, __LINE__)
#define __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, x, y, z) simt::mfma<1>((float)(a), (float)(b), c, __LINE__)
