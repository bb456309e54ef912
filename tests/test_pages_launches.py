"""What the entry points of the paged cache launch, without a device (the stand-in runtime of test_kv8_launches.py)."""
import json
import subprocess
import sys

import pytest

from test_kv8_launches import PKG, STAND_IN

CHILD = r"""
import ctypes, json, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
shim.stand_in.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_int]
sys.path.insert(0, sys.argv[3])
import moert
path, results = sys.argv[2].encode(), []
for c in json.load(open(sys.argv[4])):
    shim.stand_in(path, c.get("fail", -1), c.get("stale", 0))
    shim.stand_in_device(c.get("device", 0))
    pg = moert.Pages(*c["cache"], {n[:-4]: 0x10000 for n, _ in moert.moert_pages._fields_[7:]},
                     dtype=c.get("dtype", moert.F16))
    call = dict(c["kw"])
    if c["call"] in ("attend", "prompt"):
        call.update(q=0x20000, out=0x30000, ws=0x40000, scale=0.125)
        if "room" in call:
            call["ws_bytes"] = pg.workspace(call["heads"], call.pop("room"))
        else:
            call.setdefault("ws_bytes", 1 << 62)
        if c["call"] == "prompt":
            call.setdefault("starts", 0x50000)
    elif c["call"] == "append":
        call.update(k=0x20000, v=0x30000, slots=0x40000)
    elif c["call"] == "plan":
        call.update(new=0x20000, starts=0x30000, slots=0x40000, positions=0x50000)
    shim.stand_in_end()
    before = len(open(path).read().split("\n")) - 1
    try:
        getattr(pg, c["call"])(**call)
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
    d = tmp_path_factory.mktemp("pages_launches")
    (d / "stand_in.c").write_text(STAND_IN)
    (d / "child.py").write_text(CHILD)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-w", "-o", str(d / "stand_in.so"), str(d / "stand_in.c")], check=True)

    def run(cases):
        (d / "cases.json").write_text(json.dumps(cases))
        r = subprocess.run([sys.executable, str(d / "child.py"), str(d / "stand_in.so"), str(d / "calls"), PKG,
                            str(d / "cases.json")], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr
        return json.loads(r.stdout.strip().split("\n")[-1])

    return run


# sequences, KV heads, head dim, page, pages, pages of a sequence
def case(call, cache=(4, 8, 64, 64, 500, 100), fail=-1, stale=0, **kw):
    return dict(call=call, cache=cache, fail=fail, stale=stale, kw=kw)


def kinds(result):
    return [next(k for k in ("clear", "plan", "slots", "append", "cols", "tiles", "join_few", "join")
                 if "k_pages_" + k in line[0]) for line in result[1]]


# every form of a call: its arguments and the kernels it takes
FORMS = [
    (case("clear"), ["clear"]),
    (case("plan", tokens=9), ["plan"]),
    (case("plan", tokens=0), ["plan"]),
    (case("plan", tokens=4097), ["plan", "slots"]),
    (case("plan", cache=(1025, 1, 64, 64, 500, 100), tokens=9), ["plan", "slots"]),
    (case("append", tokens=1), ["append"]),
    (case("append", tokens=5000), ["append"]),
    (case("attend", heads=16, tokens=4), ["cols", "join_few"]),
    (case("attend", cache=(4, 1, 64, 64, 500, 100), heads=4, tokens=4), ["cols", "join"]),
    (case("attend", cache=(4, 8, 64, 64, 500, 40), heads=16, tokens=4), ["cols"]),
    (case("prompt", heads=16, tokens=90), ["cols", "join_few"]),
    (case("prompt", cache=(1, 1, 128, 64, 500, 100), heads=4, tokens=8), ["cols", "join"]),
    (case("prompt", heads=16, tokens=400), ["tiles", "join_few"]),
    (case("prompt", cache=(1, 1, 128, 64, 500, 200), heads=4, tokens=50), ["tiles", "join"]),
    (case("prompt", heads=16, tokens=5000), ["tiles"]),
]


def test_what_is_launched(launches):
    for (c, want), got in zip(FORMS, launches([c for c, _ in FORMS])):
        assert got[0] == 0 and kinds(got) == want, (c, got)


def test_nothing_follows_a_launch_that_failed(launches):
    cases = [(dict(c, fail=i), want[:i + 1]) for c, want in FORMS for i in range(len(want))]
    for (c, want), got in zip(cases, launches([c for c, _ in cases])):
        assert got[0] == -1 and kinds(got) == want, (c, got)


def test_an_error_of_an_earlier_call_is_not_the_launchs(launches):
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


def test_workspaces_do_for_all_that_they_are_asked_for(launches):
    """As many rows as the workspace was asked for, and fewer: the launchers count what their splits need."""
    cases = []
    for cache in ((1, 1, 64, 64, 5000, 4096), (1, 8, 128, 32, 5000, 5000), (3, 8, 64, 64, 500, 32), (64, 8, 64, 64, 500, 128),
                  (7, 2, 128, 256, 500, 512), (300, 4, 64, 32, 500, 97), (65535, 1, 64, 32, 500, 200), (2, 256, 64, 64, 900, 60)):
        for group in (1, 3, 16, 17, 64):
            heads = cache[1] * group
            for room in (1, 5, 37, 300, 1000, 5000):
                for tokens in sorted({1, room // 2 + 1, room}):
                    cases.append(case("prompt", cache=cache, heads=heads, tokens=tokens, room=room))
            cases.append(case("attend", cache=cache, heads=heads, tokens=cache[0], room=0))
            cases.append(case("attend", cache=cache, heads=heads, tokens=cache[0], room=700))
    for c, got in zip(cases, launches(cases)):
        assert got[0] == 0 and kinds(got)[0] in ("cols", "tiles"), (c, got)


def test_grids_stay_below_32_bits_of_threads(launches):
    cases = [case("plan", cache=(65535, 1, 64, 32, 1 << 25, 100), tokens=1 << 24),
             case("clear", cache=(65535, 1, 64, 32, 1 << 25, 100)),
             case("append", cache=(1, 8, 64, 32, 1 << 25, 100), tokens=1 << 24),
             case("append", cache=(1, 256, 64, 32, 1 << 22, 100), tokens=1 << 19)]
    for cache, heads, tokens in (((1, 1, 64, 64, 9, 16384), 64, 1 << 21), ((1, 256, 64, 64, 9, 16384), 16384, 1 << 13),
                                 ((65535, 16, 64, 32, 9, 9), 256, 1 << 19), ((65535, 1, 128, 32, 9, 999), 64, 1 << 21),
                                 ((65535, 16, 64, 32, 9, 9), 256, 65535)):
        cases += [case("prompt", cache=cache, heads=heads, tokens=tokens), case("attend", cache=cache, heads=heads, tokens=cache[0])]
    for c, got in zip(cases, launches(cases)):
        assert got[0] == 0, (c, got)
        for name, x, y, z, threads in got[1]:
            assert 0 < x * threads < 1 << 32 and y < 1 << 16 and z < 1 << 16, (c, name, x, y, z)
