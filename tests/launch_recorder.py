"""The order in which two threads' launches reach a stream, on the CPU.

The library runs in a process of its own against a stand-in for the HIP runtime that
records launches and starts no kernel, so no pointer is followed.  The first thread's first
launch waits for a moment, so that the other thread's call has the time to come in between
where nothing keeps it out."""
import shutil
import subprocess
import sys

import pytest

from nvjsel import _lib

RUNTIME = r"""
#include <chrono>
#include <condition_variable>
#include <map>
#include <mutex>
#include <string>

struct Dim { unsigned x, y, z; };
static std::mutex mu;
static std::condition_variable cv;
static bool begun = false, other = false;
static std::string order;
static std::map<const void*, std::string>& names() { static std::map<const void*, std::string> m; return m; }
static thread_local int me = 0;
static thread_local struct { Dim g, b; size_t lds; void* s; } cfg;

extern "C" {
void** __hipRegisterFatBinary(const void*) { static void* h; return &h; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* f, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
  names()[f] = name;
}
void __hipRegisterVar(void**, void*, char*, const char*, int, size_t, int, int) {}
int __hipPushCallConfiguration(Dim g, Dim b, size_t lds, void* s) { cfg = {g, b, lds, s}; return 0; }
int __hipPopCallConfiguration(Dim* g, Dim* b, size_t* lds, void** s) {
  *g = cfg.g; *b = cfg.b; *lds = cfg.lds; *s = cfg.s;
  return 0;
}
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipDeviceGetAttribute(int* v, int what, int) { *v = what == 74 ? 163840 : 256; return 0; }  // LDS; compute units
int hipGetLastError() { return 0; }
const char* hipGetErrorString(int) { return ""; }
int hipFuncSetAttribute(const void*, int, int) { return 0; }
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void*, int, size_t) { *n = 2; return 0; }
int hipLaunchKernel(const void* f, Dim, Dim, void**, size_t, void*) {
  std::unique_lock<std::mutex> lock(mu);
  order += (me == 1 ? "first:" : "other:") + names()[f] + " ";
  if (me == 1 && !begun) {
    begun = true;
    cv.notify_all();
    cv.wait_for(lock, std::chrono::seconds(1), [] { return other; });
  } else if (me != 1) {
    other = true;
    cv.notify_all();
  }
  return 0;
}
void i_am(int who) {
  me = who;
  std::unique_lock<std::mutex> lock(mu);
  if (who != 1) cv.wait_for(lock, std::chrono::seconds(30), [] { return begun; });
}
const char* launched() { return order.c_str(); }
}
"""

CALLS = r"""
import ctypes, sys, threading
runtime = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # its symbols come before the HIP runtime's
runtime.launched.restype = ctypes.c_char_p
lib = ctypes.CDLL(sys.argv[2])
P, I, L, Z, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float
codes = []

def run(who, call):
    runtime.i_am(who)
    name, types, args = eval(call)
    f = getattr(lib, name)
    f.argtypes = types
    codes.append(f(*args))

threads = [threading.Thread(target=run, args=(who, sys.argv[2 + who])) for who in (1, 2)]
for t in threads: t.start()
for t in threads: t.join()
print(codes)
print(runtime.launched().decode())
"""


def launches(tmp_path, first: str, other: str):
    """Two calls, each a text of (entry point, argument types, arguments): what they
    launched, in order, as (thread, kernel's name)."""
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    (tmp_path / "runtime.cc").write_text(RUNTIME)
    (tmp_path / "calls.py").write_text(CALLS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-pthread", "-o", str(tmp_path / "runtime.so"),
                    str(tmp_path / "runtime.cc")], check=True)
    r = subprocess.run([sys.executable, str(tmp_path / "calls.py"), str(tmp_path / "runtime.so"), str(_lib.LIB_PATH),
                        first, other], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    codes, order = r.stdout.splitlines()
    assert codes == "[0, 0]", r.stdout
    return [tuple(x.split(":")) for x in order.split()]
