"""What samhip_rope, samhip_cache_write, samhip_cache_read and samhip_cache_attn
refuse, on the host (no device is needed: nothing is launched), and that the
C++ host layer's calls of them compile, link and throw."""

import ctypes
import os
import subprocess

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def ref(x):
    return ctypes.byref(x)


def rope_desc(samhip, hd=64, pairs=(16, 16), positions=0x100, layout=0, spectrum=0, theta=10000.0, scale=None, version=1, axes=None):
    d = samhip.rope_desc(hd, list(pairs), positions, layout, spectrum, theta, scale)
    d.version = version
    if axes is not None:
        d.axes = axes
    return d


def test_rope(samhip):
    L = samhip.lib()

    def ok(x_type=0, y_type=0, w=256, rows=9, x=0x1000, y=0x10000, x_nb=None, y_nb=None, y_rows=None, y_w=None, **rope):
        e = {0: 4, 1: 2}
        xt = samhip.tensor_nd(x_type, (w, rows), (e.get(x_type, 4), x_nb or e.get(x_type, 4) * w), x)
        yt = samhip.tensor_nd(y_type, (y_w or w, rows if y_rows is None else y_rows), (e.get(y_type, 4), y_nb or e.get(y_type, 4) * w), y)
        return L.samhip_supports_rope(ref(rope_desc(samhip, **rope)), ref(xt), ref(yt))

    assert ok() == 1 and ok(x_type=1) == 1 and ok(y_type=1) == 1 and ok(x_nb=1028) == 1 and ok(y=0x1000) == 1 and ok(hd=2, pairs=(1,)) == 1
    assert ok(hd=256, pairs=(128,)) == 1 and ok(pairs=(1, 1, 1), layout=1, spectrum=1, theta=1.0, scale=[-1048576.0, 0.0, 1e-9]) == 1
    for bad in ({"hd": 3}, {"hd": 0}, {"hd": 258, "w": 258}, {"hd": 24}, {"pairs": (17, 16)}, {"pairs": (0, 4)}, {"pairs": (-1, 4)}, {"axes": 0}, {"axes": 4},
                {"axes": -1}, {"layout": 2}, {"layout": -1}, {"spectrum": 2}, {"theta": 0.5}, {"theta": float("nan")}, {"theta": float("inf")},
                {"scale": [float("nan"), 1.0]}, {"scale": [1.0, 2097152.0]}, {"positions": 0}, {"positions": 0x102}, {"version": 2}, {"rows": 0}, {"w": 0},
                {"w": 250}, {"x_type": 8}, {"y_type": 2}, {"x": 0}, {"x": 0x1002}, {"x_nb": 1000}, {"x_nb": 1026}, {"y_rows": 8}, {"y_w": 128},
                {"y": 0x1000, "y_type": 1}, {"y": 0x1000, "y_nb": 2048}, {"rows": 2 ** 23 + 1}, {"w": 2 ** 20 + 64}):
        assert ok(**bad) == 0, bad
    assert L.samhip_supports_rope(None, None, None) == 0
    assert L.samhip_rope(None, None, None, None) == samhip.ERR_INVALID_ARGUMENT


def cache_desc(samhip, type=2, kv_heads=4, hd=64, page=16, rows=160, requests=3, max_pages=5, pages=0x100, row_start=0x200, lens=0x300, k=0x10000,
               v=0x20000, k_nb=None, v_type=None, v_rows=None, w=None, version=1):
    width = kv_heads * hd if w is None else w
    block = {2: 18, 8: 34}
    kt = samhip.tensor_nd(type, (width, rows), (block.get(type, 2), k_nb or width // 32 * block.get(type, 64)), k)
    vt_type = type if v_type is None else v_type
    vt = samhip.tensor_nd(vt_type, (width, rows if v_rows is None else v_rows), (block.get(vt_type, 2), width // 32 * block.get(vt_type, 64)), v)
    c = samhip.kv_cache(kv_heads, hd, page, kt, vt, requests, max_pages, pages, row_start, lens)
    c.version = version
    return c


CACHES_REFUSED = [{"type": 0}, {"type": 1}, {"type": 12}, {"v_type": 8}, {"kv_heads": 0}, {"kv_heads": 4097}, {"hd": 16}, {"hd": 96}, {"hd": 256}, {"page": 0},
                  {"page": -1}, {"page": 2 ** 29}, {"rows": -1}, {"rows": 2 ** 31}, {"requests": 0}, {"requests": 2 ** 20 + 1}, {"max_pages": -1}, {"pages": 0},
                  {"pages": 0x101}, {"row_start": 0}, {"row_start": 0x202}, {"lens": 0}, {"lens": 0x301}, {"k": 0}, {"k": 0x10001}, {"v": 0}, {"k_nb": 142},
                  {"k_nb": 145}, {"v_rows": 161}, {"w": 128}, {"version": 0}]
CACHES_TAKEN = [{}, {"type": 8}, {"rows": 0, "k": 0, "v": 0}, {"max_pages": 0, "pages": 0}, {"k_nb": 146}, {"page": 2 ** 30, "max_pages": 1}, {"page": 1},
                {"hd": 32}, {"hd": 128}]


def test_cache_rows(samhip):
    L = samhip.lib()

    def rows(w=256, n=9, type=0, k=0x100000, v=0x200000, nb=None, v_n=None, v_type=None, v_w=None):
        e = lambda t: 2 if t == 1 else 4  # noqa: E731
        vt = type if v_type is None else v_type
        return (samhip.tensor_nd(type, (w, n), (e(type), nb or e(type) * w), k),
                samhip.tensor_nd(vt, (v_w or w, n if v_n is None else v_n), (e(vt), e(vt) * w), v))

    def write(rope=None, **t):
        k, v = rows(**t)
        return L.samhip_supports_cache_write(ref(cache_desc(samhip)), None if rope is None else ref(rope), ref(k), ref(v))

    def read(**t):
        k, v = rows(**t)
        return L.samhip_supports_cache_read(ref(cache_desc(samhip)), ref(k), ref(v))

    assert write() == 1 and read() == 1 and read(type=1) == 1 and write(rope_desc(samhip)) == 1 and write(nb=1028) == 1
    for bad in ({"w": 128}, {"n": 0}, {"n": 2 ** 23 + 1}, {"k": 0}, {"k": 0x100002}, {"v": 0}, {"nb": 1000}, {"v_n": 8}, {"v_type": 1}, {"v_w": 128},
                {"type": 8}, {"type": 26}):
        assert write(**bad) == 0 and read(**bad) == 0, bad
    assert write(type=1) == 0
    for bad in ({"hd": 32, "pairs": (8,)}, {"pairs": (33,)}, {"positions": 0}, {"version": 9}):
        assert write(rope_desc(samhip, **bad)) == 0, bad
    k, v = rows()
    for taken in CACHES_TAKEN:
        c = cache_desc(samhip, **taken)
        k, v = rows(w=c.kv_heads * c.head_dim)
        assert L.samhip_supports_cache_write(ref(c), None, ref(k), ref(v)) == 1 and L.samhip_supports_cache_read(ref(c), ref(k), ref(v)) == 1, taken
    k, v = rows()
    for bad in CACHES_REFUSED:
        c = cache_desc(samhip, **bad)
        assert L.samhip_supports_cache_write(ref(c), None, ref(k), ref(v)) == 0 and L.samhip_supports_cache_read(ref(c), ref(k), ref(v)) == 0, bad
    for call in (L.samhip_supports_cache_read, lambda c, a, b: L.samhip_supports_cache_write(c, None, a, b)):
        assert call(None, ref(k), ref(v)) == 0 and call(ref(cache_desc(samhip)), None, ref(v)) == 0 and call(ref(cache_desc(samhip)), ref(k), None) == 0
    assert L.samhip_cache_write(None, None, None, None, None) == samhip.ERR_INVALID_ARGUMENT
    assert L.samhip_cache_read(None, None, None, None) == samhip.ERR_INVALID_ARGUMENT


def test_cache_attn(samhip):
    L = samhip.lib()

    def ok(heads=8, scale=0.125, max_len=80, rows=9, q_type=0, q=0x100000, q_nb=None, w=None, out_rows=None, version=1, cache=None):
        c = cache_desc(samhip, **(cache or {}))
        width = heads * c.head_dim if w is None else w
        e = 2 if q_type == 1 else 4
        qt = samhip.tensor_nd(q_type, (width, rows), (e, q_nb or e * width), q)
        ot = samhip.tensor_nd(0, (heads * c.head_dim, rows if out_rows is None else out_rows), (4, 4 * heads * c.head_dim), 0x400000)
        d = samhip.cache_attn_desc(heads, scale, c, qt, ot, max_len)
        d.version = version
        return L.samhip_supports_cache_attn(ref(d))

    assert ok() == 1 and ok(heads=4) == 1 and ok(max_len=0) == 1 and ok(q_nb=4096) == 1 and ok(max_len=2 ** 31 - 1) == 1
    for taken in CACHES_TAKEN:
        assert ok(cache=taken) == 1, taken
    for bad in CACHES_REFUSED:
        assert ok(cache=bad) == 0, bad
    for bad in ({"heads": 6}, {"heads": 0}, {"heads": -4}, {"heads": 8192}, {"scale": float("nan")}, {"scale": float("inf")}, {"max_len": -1}, {"rows": 0},
                {"rows": 2 ** 21}, {"q_type": 1}, {"q": 0}, {"q": 0x100002}, {"q_nb": 2044}, {"w": 256}, {"out_rows": 8}, {"version": 3}):
        assert ok(**bad) == 0, bad
    assert L.samhip_supports_cache_attn(None) == 0
    assert L.samhip_cache_attn(None, None) == samhip.ERR_INVALID_ARGUMENT


SOURCE = r"""
#include "sam_hip.hpp"
#include <cstdio>
#include <stdexcept>
using namespace sam;
static void (HipBackend::*turn)(const samhip_rope_desc&, const samhip_tensor&, const samhip_tensor&) = &HipBackend::rope;
static void (HipBackend::*write)(const samhip_kv_cache&, const samhip_rope_desc*, const samhip_tensor&, const samhip_tensor&) = &HipBackend::cache_write;
static void (HipBackend::*read)(const samhip_kv_cache&, const samhip_tensor&, const samhip_tensor&) = &HipBackend::cache_read;
static void (HipBackend::*attn)(const samhip_cache_attn_desc&) = &HipBackend::cache_attn;
template <class F> static bool refused(F f) {
    try { f(); } catch (const std::invalid_argument& e) { return std::string(e.what()).find("null context") != std::string::npos; }
    return false;
}
int main() {
    samhip_rope_desc rope{};
    samhip_kv_cache cache{};
    samhip_cache_attn_desc desc{};
    samhip_tensor t{};
    const bool ok = turn && write && read && attn && refused([&] { check_status(samhip_rope(nullptr, &rope, &t, &t)); }) &&
                    refused([&] { check_status(samhip_cache_write(nullptr, &cache, nullptr, &t, &t)); }) &&
                    refused([&] { check_status(samhip_cache_read(nullptr, &cache, &t, &t)); }) &&
                    refused([&] { check_status(samhip_cache_attn(nullptr, &desc)); }) && !samhip_supports_rope(&rope, &t, &t) &&
                    !samhip_supports_cache_write(&cache, &rope, &t, &t) && !samhip_supports_cache_read(&cache, &t, &t) && !samhip_supports_cache_attn(&desc);
    std::printf("%s %zu %zu %zu\n", ok ? "ok" : "wrong", sizeof rope, sizeof cache, sizeof desc);
    return ok ? 0 : 1;
}
"""


def test_host_layer_calls(samhip, tmp_path):
    src, exe = tmp_path / "calls.cpp", tmp_path / "calls"
    src.write_text(SOURCE)
    lib = os.path.join(ROOT, "sam.cpp_amd")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(lib, "host"), str(src), "-o",
                    str(exe), "-L", lib, "-lsamhip", "-Wl,-rpath," + lib], check=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out
    sizes = [ctypes.sizeof(t) for t in (samhip.RopeDesc, samhip.KvCache, samhip.CacheAttnDesc)]
    assert out.stdout.split() == ["ok", *map(str, sizes)]   # the binding's structures are the header's


def test_division_by_page_sizes():
    """The product that stands for a division by page_rows, as the kernels take it, against the division."""
    rng = np.random.default_rng(0)
    sizes = [1, 2, 3, 5, 7, 16, 41, 48, 64, 333, 4095, 4096, 4097, 2 ** 20 + 1, 2 ** 29 - 1, 2 ** 30 - 1, 2 ** 30] + rng.integers(1, 2 ** 30, 200).tolist()
    for d in sizes:
        shift = 31 + (d - 1).bit_length()
        m = -(-(1 << shift) // d)
        assert m < 2 ** 32
        n = [0, 1, d - 1, d, d + 1, 2 ** 30, 2 ** 31 - 1, (2 ** 31 - 1) // d * d, (2 ** 31 - 1) // d * d - 1] + rng.integers(0, 2 ** 31, 200).tolist()
        for x in n:
            if 0 <= x < 2 ** 31:
                assert x * m >> shift == x // d
