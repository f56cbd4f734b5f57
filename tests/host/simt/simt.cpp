// Runs the lanes of a workgroup (hip/hip_runtime.h of this folder).
#include "hip/hip_runtime.h"

#include <sys/mman.h>

#include <map>
#include <utility>

#undef threadIdx

extern "C" void simt_swap(void** save, void* to);
// Saves the callee's registers and the stack, and goes on where `to` was saved.
asm(R"(
.text
.globl simt_swap
simt_swap:
  pushq %rbp
  pushq %rbx
  pushq %r12
  pushq %r13
  pushq %r14
  pushq %r15
  movq %rsp, (%rdi)
  movq %rsi, %rsp
  popq %r15
  popq %r14
  popq %r13
  popq %r12
  popq %rbx
  popq %rbp
  ret
)");

namespace simt {

Lane* cur;
dim3 block_idx, block_dim, grid_dim;
Wave waves[16];
void (*hook)(int) = nullptr;

namespace {
constexpr size_t kStack = 256 << 10;
Lane lanes[1024];
void* scheduler;
void (*body)(void*);
void* body_arg;

void entry() {
  body(body_arg);
  cur->done = true;
  simt_swap(&cur->sp, scheduler);
}
void stop(Stop why, int line) {
  cur->stop = why, cur->line = line;
  simt_swap(&cur->sp, scheduler);
}
// Runs the lanes [lo, hi) of one wave until they are done or at a barrier.
bool run_wave(int lo, int hi) {
  bool ran = false;
  for (;;) {
    for (int i = lo; i < hi; ++i)
      if (!lanes[i].done && lanes[i].stop == kRuns) {
        cur = &lanes[i], ran = true;
        simt_swap(&scheduler, cur->sp);
      }
    int ops = 0, others = 0;
    const Lane* first = nullptr;
    for (int i = lo; i < hi; ++i) {
      const Lane& l = lanes[i];
      if (l.done) continue;
      if (l.stop != kWaveOp) {
        ++others;
        continue;
      }
      if (!first) first = &l;
      if (l.line != first->line) fail("lanes of a wave at different operations");
      ++ops;
    }
    if (!ops) return ran;
    if (others) fail("a cross-lane operation without some live lanes");
    memset(waves[lo / 64].live[(first->ops + 1) & 1], 0, 64);
    for (int i = lo; i < hi; ++i) lanes[i].stop = kRuns;
  }
}
}  // namespace

void fail(const char* what) {
  fprintf(stderr, "simt: %s (lane %d of workgroup %u %u %u)\n", what, cur ? cur->id : -1, block_idx.x,
          block_idx.y, block_idx.z);
  abort();
}
void wave_op(int line) {
  stop(kWaveOp, line);
  ++cur->ops;
}
void barrier(int line) { stop(kBarrier, line); }

void run_block(void (*fn)(void*), void* arg, int threads) {
  body = fn, body_arg = arg;
  for (int i = 0; i < threads; ++i) {
    Lane& l = lanes[i];
    if (!l.stack) l.stack = static_cast<char*>(aligned_alloc(64, kStack));
    void** sp = reinterpret_cast<void**>(l.stack + kStack - 64);
    *--sp = nullptr, *--sp = reinterpret_cast<void*>(entry);
    for (int k = 0; k < 6; ++k) *--sp = nullptr;
    l.sp = sp, l.done = false, l.stop = kRuns, l.ops = 0, l.id = i, l.tid = dim3(i, 0, 0);
  }
  memset(waves, 0, sizeof waves);
  for (;;) {
    bool ran = false;
    for (int lo = 0; lo < threads; lo += 64) ran |= run_wave(lo, lo + 64 < threads ? lo + 64 : threads);
    const Lane* first = nullptr;
    for (int i = 0; i < threads; ++i) {
      if (lanes[i].done) continue;
      if (!first) first = &lanes[i];
      if (lanes[i].line != first->line) fail("waves at different barriers");
    }
    if (!first) return;
    if (!ran) fail("no lane can run");
    for (int i = 0; i < threads; ++i) lanes[i].stop = kRuns;
  }
}

}  // namespace simt

// An allocation's end lies before pages that cannot be touched, its start behind
// others (16 bytes of slack at most: allocations stay 16-byte aligned); its bytes
// are no zeros.
namespace {
constexpr size_t kPage = 4096, kGuard = 1 << 20;
std::map<void*, std::pair<void*, size_t>> blocks;
}  // namespace

extern "C" {
void* simt_alloc(size_t n) {
  const size_t held = (n + 15) / 16 * 16, pages = (held + kPage - 1) / kPage * kPage;
  const size_t all = kGuard + pages + kGuard;
  void* map = mmap(nullptr, all, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
  if (map == MAP_FAILED) return nullptr;
  char* p = static_cast<char*>(map) + kGuard;
  if (mprotect(p, pages, PROT_READ | PROT_WRITE)) return nullptr;
  memset(p, 0x5B, pages);
  p += pages - held;
  blocks[p] = {map, all};
  return p;
}
void simt_free(void* p) {
  const auto b = blocks.find(p);
  if (b == blocks.end()) return;
  munmap(b->second.first, b->second.second);
  blocks.erase(b);
}
void simt_hook(void (*h)(int)) { simt::hook = h; }
}
