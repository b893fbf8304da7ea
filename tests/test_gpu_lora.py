"""samhip_lora_add against its definition in F64.

Tolerance, for every element, from the arithmetic: all products and sums are
F32, so t = A x is off by at most g(K) |A||x| and y by at most
  g(K + R + 16) |scale| |B| |A| |x| + 2 u |y|,   g(n) = n u / (1 - n u), u = 2^-24
(16: the K splits' partial sums, the scale and the addition of base)."""

import ctypes

import numpy as np
import pytest

try:
    import torch
except ImportError:   # pragma: no cover
    torch = None


def describe(samhip, t):
    return samhip.tensor_nd(samhip.F16 if t.dtype == torch.float16 else samhip.F32, t.shape[::-1],
                            [v * t.element_size() for v in t.stride()[::-1]], t.data_ptr())


def strided(t, pad, dtype=None):
    dtype = dtype or t.dtype
    held = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), device=t.device, dtype=dtype)
    held[..., :t.shape[-1]] = t
    return held[..., :t.shape[-1]]


def definition(x, a, b, ids, ranks, scales, base):
    """(y, the elementwise bound) in F64."""
    m, n, slots = x.shape[0], b.shape[1], a.shape[0]
    y = torch.zeros(m, n, device=x.device, dtype=torch.float64) if base is None else base.double().clone()
    mag = torch.zeros_like(y)
    for s in range(slots):
        rows = (ids == s).nonzero()[:, 0]
        r = a.shape[1] if ranks is None else max(0, min(int(ranks[s]), a.shape[1]))
        f = 1.0 if scales is None else float(scales[s])
        aa, bb, xx = a[s, :r].double(), b[s, :, :r].double(), x[rows].double()
        y[rows] += f * ((xx @ aa.t()) @ bb.t())
        mag[rows] = abs(f) * ((xx.abs() @ aa.abs().t()) @ bb.abs().t())
    u = 2.0 ** -24
    terms = (x.shape[1] + a.shape[1] + 16) * u
    return y, terms / (1 - terms) * mag + 2 * u * y.abs() + 1e-37


def check(samhip, ctx, x, a, b, ids, ranks, scales, base, y, same=False):
    bank = samhip.lora_bank(describe(samhip, a), describe(samhip, b), None if ranks is None else ranks.data_ptr(),
                            None if scales is None else scales.data_ptr())
    ref, bound = definition(x, a, b, ids, ranks, scales, base)
    torch.cuda.synchronize()
    ctx.lora_add(bank, describe(samhip, x), samhip.tensor(samhip.I32, x.shape[0], 1, ids.data_ptr()),
                 None if base is None else describe(samhip, base), describe(samhip, y))
    ctx.synchronize()
    err = (y.double() - ref).abs()
    assert (err <= bound).all(), (err / bound).max().item()


def ids_of(order, m, slots, g):
    if order == "one":
        return torch.full((m,), slots - 1, dtype=torch.int32, device="cuda")
    if order == "runs":
        return (torch.arange(m, device="cuda") * (slots + 1) // max(m, 1) - 1).int()   # the first run has no adapter
    if order == "none":
        return torch.full((m,), -1, dtype=torch.int32, device="cuda")
    ids = torch.randint(-1, slots + 1, (m,), generator=g, device="cuda").int()          # -1 and `slots`: no adapter
    if order == "wild" and m:
        ids[:: 3] = 2 ** 31 - 1
        ids[1:: 3] = -2 ** 31
    return ids


CASES = [(1, 32, 32, 1, 1), (1, 1, 1, 1, 1), (3, 7, 5, 3, 2), (16, 1024, 1024, 16, 40), (17, 257, 65, 17, 3), (256, 1024, 4096, 16, 8),
         (201, 256, 2048, 33, 5), (777, 1001, 1359, 40, 24), (50, 4736, 1024, 128, 4), (33, 500, 258, 129, 2), (31, 96, 127, 256, 3),
         (5184, 1024, 1024, 64, 2), (1500, 64, 4736, 8, 64), (4100, 130, 259, 130, 3), (6000, 36, 50, 4, 3000), (4097, 66, 300, 2, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", CASES)
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_lora_add(samhip, gpu_ctx, shape, dtype):
    m, k, n, r, slots = shape
    print(f"lora {shape} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(m + k)
    dt = torch.float16 if dtype == "f16" else torch.float32
    for order, pad in (("runs", 0), ("scattered", 0), ("one", 3), ("none", 1), ("wild", 5)):
        x = strided(torch.randn(m, k, device="cuda", generator=g), pad)
        a = strided(torch.randn(slots, r, k, device="cuda", generator=g), pad, dt)
        b = strided(torch.randn(slots, n, r, device="cuda", generator=g), pad, dt)
        ids = ids_of(order, m, slots, g)
        ranks = torch.randint(-1, r + 3, (slots,), device="cuda", generator=g).int() if order != "one" else None
        scales = torch.randn(slots, device="cuda", generator=g) if order != "runs" else None
        if ranks is not None:   # what a slot holds behind its rank is not read
            for s, q in enumerate(ranks.clamp(0, r).tolist()):
                a[s, q:] = float("nan")
                b[s, :, q:] = float("nan")
        base = strided(torch.randn(m, n, device="cuda", generator=g), pad)
        held = torch.full((m, n + pad), 7.0, device="cuda")
        check(samhip, gpu_ctx, x, a, b, ids, ranks, scales, base, held[:, :n])
        assert (held[:, n:] == 7.0).all()
        if order in ("scattered", "wild"):
            check(samhip, gpu_ctx, x, a, b, ids, ranks, scales, None, held[:, :n])
            own = base.clone() if pad else base
            keep = own.clone()
            ref, bound = definition(x, a, b, ids, ranks, scales, keep)
            bank = samhip.lora_bank(describe(samhip, a), describe(samhip, b), ranks.data_ptr(), scales.data_ptr())
            torch.cuda.synchronize()
            gpu_ctx.lora_add(bank, describe(samhip, x), samhip.tensor(samhip.I32, m, 1, ids.data_ptr()),
                             describe(samhip, own), describe(samhip, own))
            gpu_ctx.synchronize()
            assert ((own.double() - ref).abs() <= bound).all()
            bare = (ids < 0) | (ids >= slots)
            assert torch.equal(own[bare], keep[bare])   # untouched, to the bit


@pytest.mark.gpu
def test_wide_range_of_magnitudes(samhip, gpu_ctx):
    """Values from 1e-30 to 1e30 in one row: F32 range throughout."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(40, 320, device="cuda", generator=g) * 10.0 ** torch.randint(-15, 16, (40, 1), device="cuda", generator=g)
    a = torch.randn(2, 12, 320, device="cuda", generator=g) * 1e-15
    b = torch.randn(2, 64, 12, device="cuda", generator=g) * 1e15
    ids = (torch.arange(40, device="cuda") % 2).int()
    check(samhip, gpu_ctx, x, a, b, ids, None, None, None, torch.empty(40, 64, device="cuda"))


@pytest.mark.gpu
def test_a_row_of_nan_stays_alone(samhip, gpu_ctx):
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(32, 256, device="cuda", generator=g)
    a = torch.randn(1, 16, 256, device="cuda", generator=g).half()
    b = torch.randn(1, 300, 16, device="cuda", generator=g).half()
    ids = torch.zeros(32, dtype=torch.int32, device="cuda")
    x[5, 100] = float("nan")
    x[9, 3] = float("inf")
    y = torch.empty(32, 300, device="cuda")
    bank = samhip.lora_bank(describe(samhip, a), describe(samhip, b))
    torch.cuda.synchronize()
    gpu_ctx.lora_add(bank, describe(samhip, x), samhip.tensor(samhip.I32, 32, 1, ids.data_ptr()), None, describe(samhip, y))
    gpu_ctx.synchronize()
    bad = (~torch.isfinite(y)).all(1)
    assert bad[5] and bad[9] and torch.isfinite(y[[i for i in range(32) if i not in (5, 9)]]).all()


@pytest.mark.gpu
def test_captured_replays_follow_ids_and_slots(samhip, gpu_ctx):
    """Ids, ranks and a slot's adapter change between replays."""
    g = torch.Generator(device="cuda").manual_seed(8)
    m, k, n, r, slots = 70, 512, 640, 16, 6
    x, base = torch.randn(m, k, device="cuda", generator=g), torch.randn(m, n, device="cuda", generator=g)
    a = torch.randn(slots, r, k, device="cuda", generator=g).half()
    b = torch.randn(slots, n, r, device="cuda", generator=g).half()
    ids, ranks, scales = ids_of("scattered", m, slots, g), torch.full((slots,), r, dtype=torch.int32, device="cuda"), torch.rand(slots, device="cuda")
    y = torch.empty(m, n, device="cuda")
    check(samhip, gpu_ctx, x, a, b, ids, ranks, scales, base, y)
    args = (samhip.lora_bank(describe(samhip, a), describe(samhip, b), ranks.data_ptr(), scales.data_ptr()), describe(samhip, x),
            samhip.tensor(samhip.I32, m, 1, ids.data_ptr()), describe(samhip, base), describe(samhip, y))
    torch.cuda.synchronize()
    gpu_ctx.capture_begin()
    gpu_ctx.lora_add(*args)
    graph = gpu_ctx.capture_end()
    for i in range(4):
        x.normal_(generator=g)
        ids.copy_(ids_of(("runs", "scattered", "one", "wild")[i], m, slots, g))
        ranks.copy_(torch.randint(0, r + 1, (slots,), device="cuda", generator=g))
        a[i].normal_(generator=g)
        y.zero_()
        torch.cuda.synchronize()
        graph.launch()
        gpu_ctx.synchronize()
        ref, bound = definition(x, a, b, ids, ranks, scales, base)
        assert ((y.double() - ref).abs() <= bound).all(), i
    graph.destroy()


def test_refusals(samhip):
    L = samhip.lib()

    def ok(k=64, r=8, slots=3, n=48, m=10, at=1, bt=1, version=1, ne_b=None, ne_x=None, ne_base=None, ids_type=26, ids_n=None, ids_data=0x5000,
           x_nb1=None, x_type=0, y_type=0, a_nb=None, a_data=0x10000, base=True, ranks=None):
        e = 2 if at == 1 else 4
        a = samhip.tensor_nd(at, (k, r, slots), a_nb or (e, e * k, e * k * r), a_data)
        f = 2 if bt == 1 else 4
        nb = ne_b or (r, n, slots)
        b = samhip.tensor_nd(bt, nb, (f, f * nb[0], f * nb[0] * nb[1]), 0x20000)
        nx = ne_x or (k, m)
        x = samhip.tensor_nd(x_type, nx, (4, x_nb1 or 4 * nx[0]), 0x30000)
        ids = samhip.tensor_nd(ids_type, (m if ids_n is None else ids_n,), (4,), ids_data)
        nbase = ne_base or (n, m)
        bs = samhip.tensor_nd(0, nbase, (4, 4 * nbase[0]), 0x40000)
        y = samhip.tensor_nd(y_type, (n, m), (4, 4 * n), 0x50000)
        bank = samhip.lora_bank(a, b, ranks)
        bank.version = version
        return L.samhip_supports_lora_add(ctypes.byref(bank), ctypes.byref(x), ctypes.byref(ids), ctypes.byref(bs) if base else None, ctypes.byref(y))

    assert ok() == 1 and ok(at=0, bt=0) == 1 and ok(base=False) == 1 and ok(x_nb1=1024) == 1 and ok(r=256) == 1 and ok(a_nb=(2, 200, 4000)) == 1
    for bad in ({"version": 0}, {"bt": 0}, {"at": 8}, {"r": 257}, {"r": 0}, {"slots": 0}, {"m": 0}, {"n": 0}, {"k": 0}, {"ne_b": (9, 48, 3)},
                {"ne_b": (8, 47, 3)}, {"ne_b": (8, 48, 2)}, {"ne_x": (63, 10)}, {"ne_x": (64, 9)}, {"ne_base": (48, 9)}, {"ids_type": 0},
                {"ids_n": 9}, {"ids_data": 0}, {"ids_data": 0x5002}, {"x_type": 1}, {"y_type": 1}, {"x_nb1": 252}, {"a_data": 0},
                {"a_data": 0x10001}, {"a_nb": (2, 100, 4000)}, {"ranks": 0x3}, {"m": 1 << 28}):
        assert ok(**bad) == 0, bad
    assert L.samhip_supports_lora_add(None, None, None, None, None) == 0
    assert L.samhip_lora_add(None, None, None, None, None, None) == samhip.ERR_INVALID_ARGUMENT
