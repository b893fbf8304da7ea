"""samhip_group_norm against its definition in F64.

Tolerances, relative L2 over the output: F32 outputs 1e-6.  The statistics
are F64 sums rounded once (mean as two floats, 1/deviation half a step,
2^-24), and each of the five F32 steps behind (x - hi, - lo, * 1/deviation,
* w, + b) is off by at most half a step of a value no larger than a few
outputs: below 8 * 2^-24 = 5e-7; silu and erf-GELU add at most 3e-7 of the
value (gelu_erf: 2.7e-7 of erf).  F16 outputs: half a step is 2^-11 of the
value and uniform over it, 2^-11 bounds the norm (5e-4)."""

import ctypes

import numpy as np
import pytest

try:
    import torch
except ImportError:   # pragma: no cover
    torch = None

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def definition(x, groups, w, b, eps, act):
    x = x.double()
    n, p, c = x.shape
    v = x.reshape(n, p, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3), keepdim=True)
    y = ((v - mean) / torch.sqrt(var + eps)).reshape(n, p, c)
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    if act == "relu":
        y = y.clamp(min=0)
    elif act == "silu":
        y = y * torch.sigmoid(y)
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y / 2 ** 0.5))
    return y


def describe(samhip, t):
    return samhip.tensor_nd(samhip.F16 if t.dtype == torch.float16 else samhip.F32, t.shape[::-1],
                            [v * t.element_size() for v in t.stride()[::-1]], t.data_ptr())


def strided(t, pad, dtype):
    """t in a buffer whose rows are `pad` elements longer, NaN between them."""
    held = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), device=t.device, dtype=dtype)
    held[..., :t.shape[-1]] = t
    return held[..., :t.shape[-1]]


def call(samhip, ctx, x, y, groups, w, b, eps, act):
    torch.cuda.synchronize()
    ctx.group_norm(describe(samhip, x), describe(samhip, y), groups, None if w is None else w.data_ptr(),
                   None if b is None else b.data_ptr(), eps, ACTS[act])
    ctx.synchronize()


# one pixel and one channel up to maps past the one-workgroup limit (16384
# loads of 1 or 4 channels per group), odd sizes, groups of one channel, one
# group of all, more columns than a workgroup has threads
SHAPES = [(1, 1, 1, 1), (1, 1, 8, 8), (2, 3, 6, 3), (1, 1296, 256, 8), (3, 1961, 345, 15), (1, 16385, 4, 4), (2, 16385, 5, 5), (1, 5184, 256, 8),
          (2, 5000, 96, 1), (1, 300, 4096, 2), (3, 900, 1023, 3), (1, 4096, 2052, 9), (5, 777, 260, 65), (1, 65536, 1, 1), (2, 700, 4095, 7), (1500, 9, 24, 8), (1100, 3000, 6, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("types", ["f32f32", "f16f32", "f32f16", "f16f16"])
def test_group_norm(samhip, gpu_ctx, shape, types):
    n, p, c, groups = shape
    print(f"group_norm {shape} {types}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(p + c)
    dt = {"f32": torch.float32, "f16": torch.float16}
    ti, to = dt[types[:3]], dt[types[3:]]
    for i, act in enumerate(ACTS):
        pad = (0, 3, 4, 0)[i]
        x = torch.randn(n, p, c, device="cuda", generator=g) * 1.7 + torch.randn(n, 1, c, device="cuda", generator=g)
        x = strided(x, pad, ti)
        w = torch.randn(c, device="cuda", generator=g) if i != 1 else None
        b = torch.randn(c, device="cuda", generator=g) if i != 2 else None
        held = torch.full((n, p, c + pad), 7.0, device="cuda", dtype=to)
        y = held[..., :c]
        call(samhip, gpu_ctx, x, y, groups, w, b, 1e-5, act)
        ref = definition(x, groups, w, b, 1e-5, act)
        err = ((y.double() - ref).norm() / ref.norm().clamp(min=1e-30)).item()
        assert err < (1e-6 if to == torch.float32 else 5e-4) or (y.double() - ref).abs().max().item() < 1e-6, (act, err)
        assert (held[..., c:] == 7.0).all()   # nothing behind a pixel's channels


@pytest.mark.gpu
@pytest.mark.parametrize("p", [200, 40000])
def test_mean_far_above_deviation(samhip, gpu_ctx, p):
    """A mean 1000 times the deviation: F32 sums of squares would keep one
    digit of the variance.  x itself is rounded to F32 first (the reference
    takes the rounded values), so only x - mean's exactness counts."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(1, p, 32, device="cuda", generator=g) + 1000.0
    y = torch.empty_like(x)
    call(samhip, gpu_ctx, x, y, 4, None, None, 1e-5, "none")
    ref = definition(x, 4, None, None, 1e-5, "none")
    assert ((y.double() - ref).norm() / ref.norm()).item() < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("p", [64, 30000])
def test_in_place_constant_and_nan(samhip, gpu_ctx, p):
    x = torch.randn(2, p, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x[0, :, 8:16] = 3.0                 # a constant group: y = b
    x[1, p // 2, 17] = float("nan")     # one group of one image
    ref = definition(x, 8, None, None, 1e-5, "silu")
    want = torch.isnan(ref)
    call(samhip, gpu_ctx, x, x, 8, None, None, 1e-5, "silu")
    assert torch.equal(torch.isnan(x), want) and want[1, :, 16:24].all() and want.sum().item() == p * 8
    assert (x[0, :, 8:16] == 0).all()
    ok = ~want
    assert ((x[ok].double() - ref[ok]).norm() / ref[ok].norm()).item() < 1e-6


@pytest.mark.gpu
def test_captured_replays(samhip, gpu_ctx):
    """Both forms in one graph, replayed on new contents between other work."""
    g = torch.Generator(device="cuda").manual_seed(2)
    xs = [torch.randn(1, p, 128, device="cuda", generator=g) for p in (100, 30000)]
    ys = [torch.empty_like(x) for x in xs]
    for x, y in zip(xs, ys):
        call(samhip, gpu_ctx, x, y, 8, None, None, 1e-5, "relu")
    gpu_ctx.capture_begin()
    for x, y in zip(xs, ys):
        gpu_ctx.group_norm(describe(samhip, x), describe(samhip, y), 8, None, None, 1e-5, ACTS["relu"])
    graph = gpu_ctx.capture_end()
    for i in range(4):
        for x, y in zip(xs, ys):
            x.normal_(generator=g)
            y.zero_()
        torch.cuda.synchronize()
        graph.launch()
        gpu_ctx.synchronize()
        for x, y in zip(xs, ys):
            ref = definition(x, 8, None, None, 1e-5, "relu")
            assert ((y.double() - ref).norm() / ref.norm()).item() < 1e-6
        big = torch.randn(1, 60000, 256, device="cuda", generator=g)   # scratch grows while the graph lives
        out = torch.empty_like(big)
        call(samhip, gpu_ctx, big, out, 8, None, None, 1e-5, "none")
    graph.destroy()


def sum_in_steps(t):
    """Sums over the first dimension, of at most 256 terms at once: torch's one
    sum over many blocks of F64 has lost a block's part here now and then."""
    while t.shape[0] > 1:
        t = torch.nn.functional.pad(t, (0, 0) * (t.dim() - 1) + (0, -t.shape[0] % 256)) if t.shape[0] > 256 else t
        t = t.view(-1, min(t.shape[0], 256), *t.shape[1:]).sum(1)
    return t[0]


def relative_error(y, x, groups, eps):
    """Of outputs without gain, bias and activation, relative L2."""
    n, p, c = x.shape
    v = x.double().reshape(n, p, groups, c // groups)
    mean = (sum_in_steps(v.sum(3).transpose(0, 1).contiguous()) * groups / (p * c))[:, None, :, None]
    var = (sum_in_steps((v - mean).square().sum(3).transpose(0, 1).contiguous()) * groups / (p * c))[:, None, :, None]
    ref = ((v - mean) / torch.sqrt(var + eps)).reshape(n * p, c)
    off, all = ((t.square().sum(1)) for t in (y.double().reshape(n * p, c) - ref, ref))
    return (sum_in_steps(off) / sum_in_steps(all)).sqrt().item()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((1, 82944, 256, 8), "f32"), ((1, 82944, 256, 8), "f16"), ((1, 40000, 345, 15), "f32"), ((2, 9000, 30, 6), "f16"),
                                         ((24, 2048, 256, 8), "f16"), ((24, 1024, 256, 8), "f32"), ((1, 900, 36, 4), "f32")])
@pytest.mark.parametrize("where", ["first", "two", "every 81st", "last"])
@pytest.mark.parametrize("large", [300.0, -1e4])
def test_outliers_wherever_they_stand(samhip, gpu_ctx, shape, dtype, where, large):
    """Values far from all others, as the first ones of a run and elsewhere.  An
    F32 run of 512 rounds its sum of squares by sqrt(512 / 3) half steps of 2^-24.5
    on average, 5.5e-7 of it; about the mean of the run's first batch of 32 or
    more that sum is at most 1.25 times the squared deviations; half of it
    reaches 1 / deviation: 3.4e-7 beside the 5e-7 of the other steps."""
    n, p, c, groups = shape
    x = torch.randn(n, p, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(torch.float16 if dtype == "f16" else torch.float32)
    x[:, {"first": slice(0, 1), "two": slice(0, 2), "every 81st": slice(0, None, 81), "last": slice(p - 1, None)}[where], ::c // groups] = large
    y = torch.empty(n, p, c, device="cuda")
    call(samhip, gpu_ctx, x, y, groups, None, None, 1e-5, "none")
    assert relative_error(y, x, groups, 1e-5) < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("p", [200, 40000])
@pytest.mark.parametrize("mean", [1e5, -3e6])
@pytest.mark.parametrize("channels", [32, 28])
def test_mean_a_million_deviations_away(samhip, gpu_ctx, p, mean, channels):
    """F64 sums of squares would keep four digits of the variance here.  The
    reference takes x as rounded to F32."""
    x = torch.randn(2, p, channels, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)) + mean
    y = torch.empty_like(x)
    call(samhip, gpu_ctx, x, y, 4, None, None, 1e-5, "none")
    assert relative_error(y, x, 4, 1e-5) < 1e-6


def test_refusals(samhip):
    def ok(ne=(64, 10, 2), nb=None, yne=None, ynb=None, xt=0, yt=0, groups=8, eps=1e-5, act=1, data=0x10000, w=None):
        e = 2 if xt == 1 else 4
        x = samhip.tensor_nd(xt, ne, nb or (e, e * ne[0], e * ne[0] * ne[1]), data)
        f = 2 if yt == 1 else 4
        yne = yne or ne
        y = samhip.tensor_nd(yt, yne, ynb or (f, f * yne[0], f * yne[0] * yne[1]), 0x900000)
        return samhip.lib().samhip_supports_group_norm(ctypes.byref(x), ctypes.byref(y), groups, w, None, eps, act)

    assert ok() == 1 and ok(xt=1) == 1 and ok(yt=1) == 1 and ok(nb=(4, 300, 4000)) == 1 and ok(groups=64) == 1 and ok(eps=0.0) == 1
    for bad in ({"groups": 7}, {"groups": 0}, {"act": 4}, {"act": -1}, {"eps": -1.0}, {"eps": float("nan")}, {"eps": float("inf")},
                {"ne": (64, 0, 2)}, {"ne": (64, 10, 0)}, {"ne": (64, 10, 2, 2)}, {"yne": (64, 11, 2)}, {"xt": 8}, {"yt": 26}, {"data": 0},
                {"data": 0x10002}, {"nb": (8, 512, 5120)}, {"nb": (4, 252, 2560)}, {"nb": (4, 258, 2580)}, {"nb": (4, 256, 2000)},
                {"ne": (8192, 2, 1)}, {"ne": (64, 1, 70000)}, {"w": 0x10002}):
        assert ok(**bad) == 0, bad
    x = samhip.tensor(samhip.F32, 64, 10, 0x10000)
    assert samhip.lib().samhip_supports_group_norm(None, ctypes.byref(x), 8, None, None, 1e-5, 0) == 0
    assert samhip.lib().samhip_group_norm(None, ctypes.byref(x), ctypes.byref(x), 8, None, None, 1e-5, 0) == samhip.ERR_INVALID_ARGUMENT
