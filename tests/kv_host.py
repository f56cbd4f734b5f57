"""The K/V cache's kernels and calls built for the CPU (tests/host/simt): `lib()`
is what pywelvet's lib() is for them, `Hip` has device memory on the host.

A wild access meets a guard page and ends the process: what could make one runs
in a process of its own (`run`).
"""
import ctypes
import functools
import os
import re
import subprocess
import sys
import tempfile

import numpy as np

import pywelvet as pw

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
SIMT = os.path.join(ROOT, "tests", "host", "simt")
CSRC = os.path.join(ROOT, "welvet.cuda_amd", "csrc")
CLANG = "/opt/rocm/llvm/bin/clang++"

ABI_HEAD = """
#include <cmath>
#include <cstdio>
#include <memory>
#include <string>
#include "kvcache.h"
#include "welvet_c.h"
using wv::Status;
struct welvet_kv_session {
  struct {
    void* s = nullptr;
    Status create() { return Status::ok(); }
  } stream;
  wv::KvCache cache;
};
static welvet_status to_c(const Status& s) {
  welvet_status r{};
  r.code = s.code;
  snprintf(r.message, sizeof r.message, "%s", s.message.c_str());
  return r;
}
static welvet_status invalid(const char* m) { return to_c(Status::err(wv::kInvalid, m)); }
template <class F>
welvet_status guarded(F f) { return to_c(f()); }
static void* pick(void* a, void* b) { return a ? a : b; }
namespace wv { Status init_device() { return Status::ok(); } }
extern "C" {
"""


def read(*path):
    with open(os.path.join(*path)) as f:
        return f.read()


def build(to):
    kernels = read(CSRC, "kvcache.hip")
    kernels = re.sub(r"(\bk_\w+(?:<[^<>;]*>)?)<<<(.*?)>>>\(", r"simt::launch(&\1, \2)(", kernels, flags=re.S)
    kernels = kernels.replace('asm volatile("" : "+v"(qoff));', "")
    abi = read(CSRC, "c_abi.cpp")
    abi = abi[abi.index("welvet_status welvet_kv_mount("):abi.index("// Whether an attention layer and a cache have")]
    out = os.path.join(to, "kv_host.so")
    jobs = []
    for name, text in (("kernels", kernels), ("abi", ABI_HEAD + abi + "}\n"), ("simt", read(SIMT, "simt.cpp"))):
        src = os.path.join(to, name + ".cpp")
        with open(src, "w") as f:
            f.write(text)
        jobs.append(subprocess.Popen([CLANG, "-O2", "-std=c++17", "-fPIC", "-w", "-I" + SIMT, "-I" + CSRC,
                                      "-I" + os.path.join(ROOT, "include"), "-c", src, "-o", src + ".o"]))
    for j in jobs:
        if j.wait():
            raise RuntimeError("the K/V cache's kernels do not build for the CPU")
    subprocess.check_call([CLANG, "-shared"] + [os.path.join(to, n + ".cpp.o") for n in ("kernels", "abi", "simt")]
                          + ["-o", out])
    return out


@functools.lru_cache(None)
def path():
    """The built library: given by the process that built it, or built here."""
    return os.environ.get("KV_HOST_LIB") or build(tempfile.mkdtemp(prefix="kv_host"))


HOOK = ctypes.CFUNCTYPE(None, ctypes.c_int)


@functools.lru_cache(None)
def lib():
    h = ctypes.CDLL(path())
    real = pw.lib()
    for name in ("mount", "release", "get_buffers", "append_device", "read_device", "attend_device",
                 "choose_device", "compact_device", "advance_device"):
        f, like = getattr(h, "welvet_kv_" + name), getattr(real, "welvet_kv_" + name)
        f.restype, f.argtypes = like.restype, like.argtypes
    h.simt_alloc.restype, h.simt_alloc.argtypes = ctypes.c_void_p, [ctypes.c_size_t]
    h.simt_free.restype, h.simt_free.argtypes = None, [ctypes.c_void_p]
    h.simt_hook.restype, h.simt_hook.argtypes = None, [HOOK]
    return h


def use():
    """From here on pywelvet's K/V caches are the CPU's; returns their Hip."""
    host = lib()
    pw.lib = lambda: host
    return Hip()


def run(code):
    """Runs Python code over the CPU's caches in a process of its own: `hip`, `km`
    (kv_model), `kh` (this file), `np`, `pw`, `ctypes`. Returns the process."""
    head = ("import sys, ctypes; sys.path[:0] = %r\nimport numpy as np, pywelvet as pw, kv_model as km, kv_host as kh\n"
            "hip = kh.use()\n" % ([os.path.join(ROOT, "welvet.cuda_amd"), os.path.join(ROOT, "tests")],))
    return subprocess.run([sys.executable, "-c", head + code], env=dict(os.environ, KV_HOST_LIB=path()),
                          capture_output=True, text=True, timeout=600)


class Hip:
    """pywelvet.Hip over host memory; work is done when a call returns."""

    def malloc(self, n):
        return lib().simt_alloc(int(n))

    def free(self, p):
        lib().simt_free(p)

    def upload(self, a):
        p = self.malloc(np.asarray(a).nbytes)
        self.copy_in(p, a)
        return p

    def copy_in(self, p, a):
        a = np.ascontiguousarray(a)
        ctypes.memmove(p, a.ctypes.data, a.nbytes)

    def download(self, p, shape, dtype=np.float32):
        out = np.empty(shape, dtype)
        ctypes.memmove(out.ctypes.data, p, out.nbytes)
        return out

    def memset(self, p, v, n):
        ctypes.memset(p, v, n)

    def sync(self):
        pass

    def hook(self, fn):
        """fn(0) before every launch, fn(1) before every workgroup; None ends it."""
        self.held = HOOK(fn) if fn else HOOK(0)
        lib().simt_hook(self.held)
