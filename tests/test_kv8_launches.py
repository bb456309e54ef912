"""What the entry points of the 8-bit cache launch, without a device: a stand-in for the few runtime calls they make is
loaded before the library, in a process of its own. It keeps the kernels' names and grids, and fails where it is told."""
import json
import os
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lastro-rust_amd")

STAND_IN = r"""
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>
typedef struct { uint32_t x, y, z; } dim3;
static struct { const void* f; char name[256]; } known[4096];
static int n_known, last, launches, fail_at = -1, device, at_device;
static dim3 g, b;
static size_t shm;
static void* stream;
static FILE* out;
void stand_in(const char* path, int fail, int stale) {
  if (!out) out = fopen(path, "w");
  launches = 0, fail_at = fail, last = stale;
}
void stand_in_end(void) { fflush(out); }
void** __hipRegisterFatBinary(const void* d) { static void* m; return &m; }
void __hipUnregisterFatBinary(void** m) {}
void __hipRegisterVar(void** m, void* v, char* h, char* d, int e, size_t s, int c, int q) {}
void __hipRegisterFunction(void** m, const void* f, char* d, const char* name, unsigned t, void* ti, void* bi, dim3* bd,
                           dim3* gd, int* w) {
  if (n_known == 4096) return;
  known[n_known].f = f;
  strncpy(known[n_known++].name, name, 255);
}
int __hipPushCallConfiguration(dim3 grid, dim3 block, size_t s, void* st) { g = grid, b = block, shm = s, stream = st; return 0; }
int __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* s, void** st) { *grid = g, *block = b, *s = shm, *st = stream; return 0; }
int hipLaunchKernel(const void* f, dim3 grid, dim3 block, void** a, size_t s, void* st) {
  const char* name = "?";
  for (int i = 0; i < n_known; i++) if (known[i].f == f) name = known[i].name;
  fprintf(out, "%s %u %u %u %u\n", name, grid.x, grid.y, grid.z, block.x);
  if (launches++ == fail_at) return last = 9;
  return 0;
}
int hipGetLastError(void) { const int e = last; last = 0; return e; }
const char* hipGetErrorString(int e) { return "told to fail"; }
void stand_in_device(int d) { at_device = d; }
int hipGetDevice(int* d) { *d = device; return 0; }
int hipSetDevice(int d) { device = d; fprintf(out, "device %d 0 0 0\n", d); return 0; }
/* type (2: device memory), device, then pointers */
int hipPointerGetAttributes(int* a, const void* p) { memset(a, 0, 16); a[0] = 2; a[1] = at_device; return 0; }
"""

CHILD = r"""
import ctypes, json, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
shim.stand_in.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_int]
sys.path.insert(0, sys.argv[3])
import moert
path, cases, results = sys.argv[2].encode(), json.loads(sys.argv[4]), []
for c in cases:
    shim.stand_in(path, c.get("fail", -1), c.get("stale", 0))
    shim.stand_in_device(c.get("device", 0))
    at = {n[:-4]: 0x10000 for n, _ in moert.moert_kv8._fields_[4:]}
    kv = moert.Kv8(*c["cache"], at)
    call = dict(c["kw"])
    if c["call"] == "attend":
        call.update(q=0x20000, out=0x30000, ws=0x40000, ws_bytes=1 << 62, scale=0.125)
    elif c["call"] in ("append", "read"):
        call.update(k=0x20000, v=0x30000)
    shim.stand_in_end()
    before = len(open(path).read().split("\n")) - 1
    try:
        getattr(kv, c["call"])(**call)
        code = 0
    except moert.MoertError as e:
        code = e.code
    shim.stand_in_end()
    lines = open(path).read().split("\n")[before:-1]
    results.append([code, [[l.split()[0]] + [int(x) for x in l.split()[1:]] for l in lines]])
print(json.dumps(results))
"""


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv8_launches")
    (d / "stand_in.c").write_text(STAND_IN)
    (d / "child.py").write_text(CHILD)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-w", "-o", str(d / "stand_in.so"), str(d / "stand_in.c")], check=True)

    def run(cases):
        r = subprocess.run([sys.executable, str(d / "child.py"), str(d / "stand_in.so"), str(d / "calls"), PKG,
                            json.dumps(cases)], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr
        return json.loads(r.stdout.strip().split("\n")[-1])

    return run


def case(call, cache=(2, 8, 64, 4096), fail=-1, stale=0, **kw):
    return dict(call=call, cache=cache, fail=fail, stale=stale, kw=kw)


def kinds(result):
    return [next(k for k in ("clear", "append", "advance", "attend", "combine", "finish", "mass", "read", "evict")
                 if "k_kv8_" + k in line[0]) for line in result[1]]


# every form of a call: its arguments and the kernels it takes
FORMS = [
    (case("clear"), ["clear"]),
    (case("append", n=1), ["append"]),
    (case("append", n=4000), ["append", "advance"]),
    (case("attend", heads=16, n=1), ["attend", "combine"]),
    (case("attend", cache=(2, 8, 64, 96), heads=16, n=1), ["attend"]),
    (case("attend", heads=16, n=1, mass_decay=1.0), ["attend", "finish"]),
    (case("attend", cache=(1, 1, 64, 65536), heads=16, n=20), ["attend", "combine"]),
    (case("attend", cache=(1, 1, 64, 65536), heads=16, n=20, mass_decay=0.5), ["attend", "combine", "mass"]),
    (case("attend", cache=(2, 8, 128, 96), heads=32, n=9, mass_decay=0.5), ["attend", "mass"]),
    (case("evict", keep=4), ["evict"]),
    (case("read", pos=0, n=9), ["read"]),
]


def test_what_is_launched(launches):
    for (c, want), got in zip(FORMS, launches([c for c, _ in FORMS])):
        assert got[0] == 0 and kinds(got) == want, (c, got)


def test_nothing_follows_a_launch_that_failed(launches):
    """What comes behind a launch reads what that one was to write: lengths do not move on without rows, and no mass is
    made of a workspace that no attention has written."""
    cases = [(dict(c, fail=i), want[:i + 1]) for c, want in FORMS for i in range(len(want))]
    for (c, want), got in zip(cases, launches([c for c, _ in cases])):
        assert got[0] == -1 and kinds(got) == want, (c, got)


def test_grids_stay_below_32_bits_of_threads(launches):
    shapes = [((1, 1, 64, 1 << 20), 64, 1 << 20), ((2, 1, 64, 1 << 20), 32, 1 << 20), ((1, 2, 128, 1 << 20), 64, 1 << 20),
              ((9, 1, 64, 1 << 20), 14, 1 << 20), ((65535, 16, 64, 96), 1024, 2), ((1, 256, 64, 1 << 20), 16384, 1 << 13)]
    cases = [case("attend", cache=c, heads=heads, n=n, mass_decay=decay) for c, heads, n in shapes
             for decay in (None, 1.0)]
    for c, got in zip(cases, launches(cases)):
        assert got[0] == 0 and kinds(got)[0] == "attend", (c, got)
        for name, x, y, z, threads in got[1]:
            assert x * threads < 1 << 32 and y < 1 << 16 and z < 1 << 16, (c, name, x, y, z)


def test_an_error_of_an_earlier_call_is_not_the_launchs(launches):
    """The runtime keeps a thread's last error until it is asked for. One that the caller has dealt with (an allocation
    that did not fit, say) makes no call fail, and leaves none half done."""
    for (c, want), got in zip(FORMS, launches([dict(c, stale=2) for c, _ in FORMS])):
        assert got[0] == 0 and kinds(got) == want, (c, got)


def test_calls_run_on_the_buffers_device_and_leave_the_current_one(launches):
    """Also where a launch fails."""
    for fail in (-1, 0):
        for (c, want), got in zip(FORMS, launches([dict(c, device=3, fail=fail) for c, _ in FORMS])):
            lines = [(line[0], line[1]) for line in got[1]]
            assert lines[0] == ("device", 3) and lines[-1] == ("device", 0), (c, got)
            assert len(lines) == 2 + (len(want) if fail < 0 else 1) and got[0] == (0 if fail < 0 else -1), (c, got)
            assert all(name != "device" for name, _ in lines[1:-1]), (c, got)
