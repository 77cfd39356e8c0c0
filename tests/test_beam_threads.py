"""Selections of two threads on one stream, which share a workspace.

CPU: the order in which their launches reach the stream.  The library runs in a process of its own against a stand-in for the HIP runtime that
records launches and starts no kernel.  Its scan launch waits for a moment, so
that another thread's call, which may use the same workspace, has the time to come
between a scan and the join that reads what the scan wrote.  GPU: the results of many calls
that two threads queue without waiting for any."""
import shutil
import subprocess
import sys
import threading

import pytest
import torch

import nvjsel
from nvjsel import _lib

RUNTIME = r"""
#include <condition_variable>
#include <chrono>
#include <cstring>
#include <map>
#include <mutex>
#include <string>

struct Dim { unsigned x, y, z; };
static std::mutex mu;
static std::condition_variable cv;
static bool scanned = false, other = false;
static std::string order;
static std::map<const void*, std::string>& names() { static std::map<const void*, std::string> m; return m; }
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
int hipDeviceGetAttribute(int* v, int, int) { *v = 256; return 0; }
int hipGetLastError() { return 0; }
int hipLaunchKernel(const void* f, Dim, Dim, void**, size_t, void*) {
  const std::string& n = names()[f];
  std::unique_lock<std::mutex> lock(mu);
  if (n.find("beam_scan_kernel") != std::string::npos) {
    order += "scan ";
    scanned = true;
    cv.notify_all();
    cv.wait_for(lock, std::chrono::seconds(1), [] { return other; });
  } else if (n.find("beam_join_kernel") != std::string::npos) {
    order += "join ";
  } else {
    order += "one ";
    other = true;
    cv.notify_all();
  }
  return 0;
}
void wait_scanned() {
  std::unique_lock<std::mutex> lock(mu);
  cv.wait_for(lock, std::chrono::seconds(30), [] { return scanned; });
}
const char* launched() { return order.c_str(); }
}
"""

CALLS = r"""
import ctypes, sys, threading
runtime = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # its symbols come before the HIP runtime's
runtime.launched.restype = ctypes.c_char_p
lib = ctypes.CDLL(sys.argv[2])
p, i, l, z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
lib.nvjsel_beam_select.argtypes = [p, i, i, i, i, l, l, p, p, i, i, p, p, p, p, z, p]

def select(batch, beams, vocab):  # nothing is launched: no pointer is followed
    at = 0x1000
    return lib.nvjsel_beam_select(at, 1, batch, beams, vocab, beams * vocab, vocab, at, None, 0, 8, at, at, at, at, 1 << 40, None)

codes = []
large = threading.Thread(target=lambda: codes.append(select(24, 8, 20011)))
def small():
    runtime.wait_scanned()
    codes.append(select(2, 4, 9001))
other = threading.Thread(target=small)
large.start(), other.start(), large.join(), other.join()
print(codes, runtime.launched().decode())
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_no_call_comes_between_a_scan_and_its_join(tmp_path):
    (tmp_path / "runtime.cc").write_text(RUNTIME)
    (tmp_path / "calls.py").write_text(CALLS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-pthread", "-o", str(tmp_path / "runtime.so"),
                    str(tmp_path / "runtime.cc")], check=True)
    r = subprocess.run([sys.executable, str(tmp_path / "calls.py"), str(tmp_path / "runtime.so"), str(_lib.LIB_PATH)],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split(" ", 2)[:2] == ["[0,", "0]"], r.stdout
    assert r.stdout.split()[2:] == ["scan", "join", "one"], r.stdout


@pytest.mark.gpu
def test_two_threads_queue_small_and_large_selections():
    g = torch.Generator().manual_seed(3)
    shapes = [(2, 4, 9001), (24, 8, 20011)]  # of one launch, and of two
    data = [((torch.randn(b, w, v, generator=g) * 2).to(torch.bfloat16).cuda(), torch.randn(b, w, generator=g).cuda())
            for b, w, v in shapes]
    want = [nvjsel.beam_search_select(*x, num_candidates=8) for x in data]
    torch.cuda.synchronize()
    got = [[], []]
    start = threading.Barrier(2)

    def queue(at):
        start.wait()
        for _ in range(100):
            got[at].append(nvjsel.beam_search_select(*data[at], num_candidates=8))

    threads = [threading.Thread(target=queue, args=(at,)) for at in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for at in range(2):
        assert len(got[at]) == 100
        assert all(torch.equal(a, b) for out in got[at] for a, b in zip(out, want[at]))
