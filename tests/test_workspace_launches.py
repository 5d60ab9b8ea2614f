"""The launches of a call stay together on its workspace.

Calls from several threads on one stream share the stream's workspace.  Some
calls are two launches, the second of which reads what the first left in the
workspace, so no launch of another call with that workspace may come between
them.  Here the HIP runtime's launch functions are replaced, in a process of
their own, by ones that write down the order of launches and take their time;
nothing reaches a GPU."""

import itertools
import json
import os
import shutil
import subprocess
import sys

import pytest

from sglang_mlx_amd import _lib

CC = shutil.which("cc") or shutil.which("gcc")

STUB = r"""
#include <pthread.h>
#include <stddef.h>
#include <unistd.h>
typedef struct { unsigned x, y, z; } dim3;
static pthread_mutex_t mu = PTHREAD_MUTEX_INITIALIZER;
static int order[65536], launches;
static __thread int call;
static __thread dim3 grid, block;
static __thread size_t shared;
static __thread void* stream;
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t n, void* s) { grid = g, block = b, shared = n, stream = s; return 0; }
int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* n, void** s) { *g = grid, *b = block, *n = shared, *s = stream; return 0; }
int hipGetLastError(void) { return 0; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipDeviceGetAttribute(int* v, int what, int d) { *v = 256; return 0; }
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, const void* f, int t, size_t s) { *n = 2; return 0; }
int hipLaunchKernel(const void* f, dim3 g, dim3 b, void** a, size_t n, void* s) {
  pthread_mutex_lock(&mu);
  if (launches < 65536) order[launches++] = call;
  pthread_mutex_unlock(&mu);
  usleep(300);
  return 0;
}
void stub_call(int i) { call = i; }
int stub_launches(void) { return launches; }
int stub_order(int i) { return order[i]; }
"""

PROGRAM = r"""
import ctypes, importlib.util, json, sys, threading
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
spec = importlib.util.spec_from_file_location("signatures", sys.argv[2])
_lib = importlib.util.module_from_spec(spec)
spec.loader.exec_module(_lib)
lib = _lib.lib()
buf = ctypes.create_string_buffer(1024)
P = (ctypes.addressof(buf) + 63) // 64 * 64  # no launch runs: never read
BF = _lib.PKV_BF16
cache = (10, 1.0, 1024, 4096, 2048, 4096, 2048)  # num_blocks, scale, strides


def extend(ws, N, B, max_query):
    return lib.pkv_paged_attention_extend(P, P, P, P, P, P, P, N, B, 8, 2, 128, 16, 1024, 16384, max_query, 0, 0,
                                          *cache, ws, 1 << 40, BF, BF, 1.0, 1.0, None)


def decode(ws, max_seq_len, layout):
    need = lib.pkv_paged_attention_workspace_size(1, 8, 2, 128, max_seq_len, 0)
    head = 2048 if layout == 0 else 128
    return lib.pkv_paged_attention(P, P, P, P, P, P, None, 1, 8, 2, 128, 16, 8192, max_seq_len, 10, 1.0, 1024, 4096, head,
                                   4096, head, layout, 0, ws, need, BF, BF, 1.0, 1.0, None)


def cascade(ws):
    plan = _lib.CascadePlanC(P, P, P, P, 2, 1, 2, 128, 2, 64, 2)
    return lib.pkv_paged_attention_cascade(P, P, P, P, P, P, None, ctypes.byref(plan), 2, 8, 2, 128, 16, 1024, 16384,
                                           *cache, ws, 1 << 40, BF, BF, 1.0, 1.0, None)


CALLS = {
    "row tiles": lambda ws: extend(ws, 20, 1, 20),
    "few rows": lambda ws: extend(ws, 2, 2, 1),
    "decode": lambda ws: decode(ws, 1024, 0),
    "partitions": lambda ws: decode(ws, 131072, 0),
    "token rows": lambda ws: decode(ws, 131072, 1),
    "cascade": cascade,
}


def run(number, names, ws):
    for i, name in enumerate(names):
        stub.stub_call(number * 1000 + i)
        st = CALLS[name](ws)
        assert st == 0, (name, lib.pkv_last_error())


if sys.argv[3] == "count":
    out = {}
    for i, name in enumerate(CALLS):
        at = stub.stub_launches()
        run(i, [name], P)
        out[name] = stub.stub_launches() - at
    print(json.dumps(out))
else:
    names = sys.argv[4].split(",")
    threads = [threading.Thread(target=run, args=(k, [name] * 40, P)) for k, name in enumerate(names)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    print(json.dumps([stub.stub_order(i) for i in range(stub.stub_launches())]))
"""

TWO = ("row tiles", "partitions", "token rows", "cascade")  # calls of two launches
ONE = ("few rows", "decode")


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    if CC is None or not os.path.exists(_lib.LIB_PATH):
        pytest.skip("no C compiler, or the library is not built")
    where = tmp_path_factory.mktemp("launches")
    (where / "stub.c").write_text(STUB)
    (where / "program.py").write_text(PROGRAM)
    stub = str(where / "stub.so")
    subprocess.run([CC, "-shared", "-fPIC", "-O1", "-o", stub, str(where / "stub.c"), "-lpthread"], check=True)

    def run(*args):
        done = subprocess.run([sys.executable, str(where / "program.py"), stub, _lib.__file__, *args], timeout=120,
                              capture_output=True, text=True)
        assert done.returncode == 0 and not done.stderr, done.stderr
        return json.loads(done.stdout)

    return run


def test_launches_of_each_call(launches):
    # (The pairs below test nothing if a call becomes one launch.)
    assert launches("count") == {**{n: 2 for n in TWO}, **{n: 1 for n in ONE}}


@pytest.mark.parametrize("pair", list(itertools.combinations_with_replacement(TWO, 2))
                         + list(itertools.product(TWO, ONE)), ids=" + ".join)
def test_no_launch_comes_between_those_of_a_call(launches, pair):
    order = launches("pair", ",".join(pair))
    runs = [call for call, _ in itertools.groupby(order)]
    assert len(runs) == 80 and len(set(runs)) == 80, "a call's launches are apart"
