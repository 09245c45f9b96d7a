"""What libamla.so asks of the HIP runtime, without a GPU: launches and LDS limits, in order.

A small library defines the runtime's launch functions and is loaded before libamla.so, in a
process of its own; nothing runs on a device and nothing reads the pointers."""
import json
import os
import shutil
import subprocess
import sys

import pytest

STUB = r"""
#include <cstddef>
#include <cstdio>
#include <string>
struct dim3_ { unsigned x, y, z; };
static thread_local struct { dim3_ g, b; size_t lds; void *st; } cfg;
static std::string log_;
extern "C" {
int __hipPushCallConfiguration(dim3_ g, dim3_ b, size_t lds, void *st) { cfg = {g, b, lds, st}; return 0; }
int __hipPopCallConfiguration(dim3_ *g, dim3_ *b, size_t *lds, void **st) {
  *g = cfg.g; *b = cfg.b; *lds = cfg.lds; *st = cfg.st;
  return 0;
}
int hipLaunchKernel(const void *f, dim3_ g, dim3_ b, void **, size_t lds, void *) {
  char t[160];
  snprintf(t, sizeof t, "[\"launch\",%llu,%u,%u,%zu],", (unsigned long long)f, g.x, b.x, lds);
  log_ += t;
  return 0;
}
int hipFuncSetAttribute(const void *f, int, int v) {
  char t[96];
  snprintf(t, sizeof t, "[\"lds\",%llu,%d],", (unsigned long long)f, v);
  log_ += t;
  return 0;
}
int hipGetLastError() { return 0; }
const char *stub_take() {
  static std::string out;
  out = "[" + log_ + "null]";
  log_.clear();
  return out.c_str();
}
}
"""

RUN = """
import ctypes, json, sys
stub = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
from amla import _lib
L = _lib.lib()
stub.stub_take.restype = ctypes.c_char_p
out = []
for name, args in json.loads(sys.stdin.read()):
    stub.stub_take()
    rc = getattr(L, name)(*args)
    out.append([rc, json.loads(stub.stub_take())[:-1]])
print("RESULT" + json.dumps(out))
"""


def hip_calls(tmp_path, calls):
    """[(entry, args)] -> [(return code, [["launch", kernel, blocks, threads, lds] | ["lds", kernel, bytes]])]."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, so = tmp_path / "stub.cpp", tmp_path / "libstub.so"
    src.write_text(STUB)
    subprocess.run([gxx, "-shared", "-fPIC", "-O1", "-o", str(so), str(src)], check=True)
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-on-one-gpu_amd")
    res = subprocess.run([sys.executable, "-c", RUN, str(so), pkg], input=json.dumps(calls), text=True,
                         capture_output=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    return json.loads(res.stdout.split("RESULT")[1])
