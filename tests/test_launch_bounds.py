"""Launches of very large calls (CPU test): HIP takes fewer than 2^32 threads in one, so log probabilities of very many rows and
AdamW over very many elements go in several.  The library runs here on a stand-in for the HIP runtime that records what
would be launched, in a process of its own; the pointers are numbers that nobody follows."""
import json
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "erfnet_pytorch_amd", "liberfnet_hip.so")

STAND_IN = r"""
#include <cstddef>
#include <cstring>
struct Dim { unsigned x, y, z; };
struct Launch { unsigned grid[3], block[3]; unsigned char argument[4096]; };
static Launch launches[64];
static int count;
static Dim grid_, block_;
static size_t lds_;
static void *stream_;
extern "C" {
int __hipPushCallConfiguration(Dim g, Dim b, size_t l, void *s) { grid_ = g; block_ = b; lds_ = l; stream_ = s; return 0; }
int __hipPopCallConfiguration(Dim *g, Dim *b, size_t *l, void **s) { *g = grid_; *b = block_; *l = lds_; *s = stream_; return 0; }
int hipLaunchKernel(const void *, Dim g, Dim b, void **args, size_t, void *)
{
    if (count < 64) {
        Launch &l = launches[count];
        const unsigned from[6] = {g.x, g.y, g.z, b.x, b.y, b.z};
        memcpy(l.grid, from, sizeof(from));
        memcpy(l.argument, args[0], bytes_of_argument);
    }
    ++count;
    return 0;
}
int hipGetLastError(void) { return 0; }
int hipStreamIsCapturing(void *, int *status) { *status = 0; return 0; }
void *__hipRegisterFatBinary(const void *) { static void *p; return &p; }
void __hipRegisterFunction(void) {}
void __hipRegisterVar(void) {}
void __hipUnregisterFatBinary(void *) {}
int launch_count(void) { return count; }
const Launch *launch(int i) { return &launches[i]; }
void forget(void) { count = 0; }
}
"""

PRELUDE = r"""
import ctypes as C, json, struct, sys
hip = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
lib = C.CDLL(sys.argv[2])
hip.launch.restype = C.POINTER(C.c_ubyte)
lib.erf_last_error.restype = C.c_char_p
lib.erf_log_probs_workspace_bytes.restype = C.c_size_t
ll, vp = C.c_longlong, C.c_void_p

def launches():
    out = []
    assert hip.launch_count() <= 64
    for i in range(hip.launch_count()):
        raw = bytes(hip.launch(i)[:24 + 4096])
        out.append((struct.unpack("6I", raw[:24]), raw[24:]))
    hip.forget()
    return out
"""


def run(tmp_path, argument_bytes, script, *args):
    """`script` behind the prelude, in a process whose HIP calls are the stand-in's; what it prints, as JSON."""
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    if not os.path.exists(LIB):
        from erfnet_pytorch_amd import _lib
        _lib.build()
    src, so = tmp_path / "hip.cpp", tmp_path / "hip.so"
    src.write_text(STAND_IN.replace("bytes_of_argument", str(argument_bytes)))
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-Wno-builtin-declaration-mismatch", str(src), "-o", str(so)], check=True, timeout=120)
    r = subprocess.run([sys.executable, "-c", PRELUDE + script, str(so), LIB, *map(str, args)], capture_output=True, text=True,
                       timeout=120, cwd="/")
    assert r.returncode == 0, r.stderr[-3000:]
    return json.loads(r.stdout.splitlines()[-1])


LOG_PROBS = r"""
outer, V, inner, k, size = (int(a) for a in sys.argv[3:8])
base = {n: (i + 1) << 48 for i, n in enumerate(("x", "target", "lp", "ent", "stats", "top", "idx", "g_lp", "g_h", "g_top", "dx", "ws"))}
p = {n: vp(a) for n, a in base.items()}
tail = "_bf16" if size == 2 else ""
ld = V + 8
n_ws = lib.erf_log_probs_workspace_bytes(ll(outer), V, ll(inner), k)
top = (p["top"], p["idx"]) if k else (None, None)
fwd = getattr(lib, "erf_log_probs_forward" + tail)
rc = fwd(p["x"], p["target"], p["lp"], p["ent"], p["stats"], *top, ll(outer), V, ll(inner), ll(ld), k, ll(-1), p["ws"],
         C.c_size_t(n_ws), None)
forward, why = launches(), lib.erf_last_error().decode()
bwd = getattr(lib, "erf_log_probs_backward" + tail)
rc2 = bwd(p["x"], p["target"], p["ent"], p["stats"], top[1], p["g_lp"], p["g_h"], p["g_top"] if k else None, p["dx"], ll(outer), V,
          ll(inner), ll(ld), k, ll(-1), None)
backward = launches()

def read(raw):      # LpDesc: 7 pointers, rows, ld, inner, group, next, ignore, V, k, splits, seg, 2 pointers, 4 pointers
    f = struct.unpack("7Q6q4i2Q3QQ", raw[:168])
    d = dict(zip(("x", "target", "lp", "ent", "stats", "top", "idx", "rows", "ld", "inner", "group", "next", "ignore", "V", "k", "splits", "seg",
                  "part", "part_keys", "g_lp", "g_h", "g_top", "dx"), f))
    return d

group = V * inner if inner > 1 else ld
step = dict(x=group * size, target=8 * inner, lp=4 * inner, ent=4 * inner, stats=8 * inner, top=4 * k * inner, idx=8 * k * inner, g_lp=4 * inner,
            g_h=4 * inner, g_top=4 * k * inner, dx=V * inner * size)
out = []
for calls in (forward, backward):
    spans = []
    for grid, raw in calls:
        d = read(raw)
        at = (d["target"] - base["target"]) // step["target"]
        moved = all(d[n] - base[n] == at * s for n, s in step.items() if d[n])
        spans.append([at, d["rows"] // inner, grid[0], grid[3], bool(moved), grid[1:3] + grid[4:]])
    out.append(spans)
print(json.dumps([rc, rc2, why] + out))
"""


@pytest.mark.parametrize("size", [2, 4])
@pytest.mark.parametrize("outer,v,inner,k", [
    (17_000_000, 1025, 1, 0), (17_000_000, 8192, 1, 3), (70_000_000, 129, 1, 8), (70_000_000, 1000, 1, 2),
    (20_000_000, 40_000, 1, 1), ((1 << 34) + 5, 20, 1, 2), ((1 << 32) + 77, 3, 1, 0), (9000, 20, 1 << 20, 2), (3, 2, (1 << 31) + 11, 1),
    (5, 131072, 1, 20), (2047, 100003, 1, 8), (6, 20, 512 * 1024, 8), (1, 1 << 30, 1, 64)])
def test_log_probs_of_any_number_of_rows_are_launched_within_hips_bounds(tmp_path, outer, v, inner, k, size):
    rc, rc2, why, forward, backward = run(tmp_path, 168, LOG_PROBS, outer, v, inner, k, size)
    assert rc == 0 and rc2 == 0, why
    joins = 1 if inner == 1 and outer <= 128 and v >= 65536 else 0
    for calls, extra in ((forward, joins), (backward, 0)):
        parts = calls[:len(calls) - extra]
        for at, n, blocks, threads, moved, rest in calls:
            assert 0 < blocks * threads < 1 << 32 and moved and rest == [1, 1, 1, 1], (blocks, threads)
        parts = sorted(c[:2] for c in parts)
        assert parts[0][0] == 0 and all(a + n == b for (a, n), (b, _) in zip(parts, parts[1:])) and sum(parts[-1]) == outer
    if outer * inner < 1 << 23:
        assert len(forward) == 1 + joins and len(backward) == 1


def test_log_probs_of_an_image_beyond_one_launch_are_refused(tmp_path):
    rc, rc2, why, forward, backward = run(tmp_path, 168, LOG_PROBS, 1, 2, (1 << 32) - 200, 1, 2)
    assert rc and rc2 and "pixels an image" in why and not forward and not backward


ADAMW = r"""
bits, size = int(sys.argv[3]), int(sys.argv[4])
sizes = json.loads(sys.argv[5])
count, most = len(sizes), 92 if bits == 8 else 126
names = ["p", "g", "m", "ms", "v", "vs"] if bits == 8 else ["p", "g", "m", "v"]
step = dict(p=size, g=size, m=1 if bits == 8 else 4, v=1 if bits == 8 else 4, ms=4 / 256, vs=4 / 256)
room = (1 << 47) // (6 * count)         # of one tensor's table entry
base = {n: [(j * count + i) * room + 256 for i in range(count)] for j, n in enumerate(names)}
table = {n: (vp * count)(*base[n]) for n in names}
name = "erf_adamw8_step" if bits == 8 else "erf_adamw_step"
rc = getattr(lib, name + ("_bf16" if size == 2 else ""))(
    count, *[table[n] for n in names], (ll * count)(*sizes), C.c_double(1e-3), C.c_double(0.9), C.c_double(0.999), C.c_double(1e-8),
    C.c_double(0.01), ll(1), None)
pointers = ["p", "g", "m", "v", "ms", "vs"][:len(names)]
out = []
for grid, raw in launches():        # AdamwDesc: 8 floats, count, end_chunk, last, low halves, pairs of upper 16 bits
    n, = struct.unpack("i", raw[32:36])
    u = struct.unpack(f"{most * (2 + len(names) + len(names) // 2)}I", raw[36:36 + 4 * most * (2 + len(names) + len(names) // 2)])
    part = lambda j: u[j * most:(j + 1) * most]
    end, last = part(0), part(1)
    for t in range(n):
        first = end[t - 1] if t else 0
        elements = (end[t] - first - 1) * 2048 + last[t]
        at = {}
        for j, name in enumerate(pointers):
            high = part(2 + len(names) + j // 2)[t] >> (16 * (j & 1)) & 0xffff
            at[name] = high << 32 | part(2 + j)[t]
        i = max(k for k in range(count) if base["p"][k] <= at["p"])
        begin = (at["p"] - base["p"][i]) // size
        moved = all(at[n] - base[n][i] == begin * s for n, s in ((n, step[n]) for n in names))
        out.append([i, begin, elements, bool(moved)])
    out.append([grid[0], grid[3], end[n - 1]])
print(json.dumps([rc, lib.erf_last_error().decode(), out]))
"""


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [2, 4])
@pytest.mark.parametrize("sizes", [
    [7], [100] * 229, [0, 5, 0, 2048, 0], [35_000_000_000], [10, 34_359_738_367 * 3, 2049], [20_000_000_000, 20_000_000_000, 3],
    [(2 ** 24 - 1) * 2048, 5], [(2 ** 24 - 1) * 2048 - 1, 5], [(2 ** 24 - 1) * 2048 + 1, 5]], ids=lambda s: f"{len(s)}x{max(s)}")
def test_adamw_of_any_number_of_elements_is_launched_within_hips_bounds(tmp_path, sizes, size, bits):
    rc, why, out = run(tmp_path, 4096, ADAMW, bits, size, json.dumps(sizes))
    assert rc == 0, why
    launches, parts = [o for o in out if len(o) == 3], [o for o in out if len(o) == 4]
    for blocks, threads, chunks in launches:
        assert blocks == chunks and 0 < blocks * threads < 1 << 32
    at = {}
    for i, begin, elements, moved in parts:
        assert moved and begin == at.get(i, 0) and begin % 2048 == 0 and elements > 0
        at[i] = begin + elements
    assert at == {i: n for i, n in enumerate(sizes) if n}
    if sum(sizes) < 1 << 30:
        assert len(launches) == -(-sum(n > 0 for n in sizes) // (92 if bits == 8 else 126))
