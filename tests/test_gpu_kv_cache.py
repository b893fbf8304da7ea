"""Rotary positions (samhip_rope), rows to and from caches of keys and values
in Q8_0 or Q4_0 pages (samhip_cache_write, samhip_cache_read) and attention over
them (samhip_cache_attn), against their definitions in F64.

Rotation.  cos and sin are F32 numbers (2^-24 each), each product and the sum
are rounded (2^-24): |error| <= 4 * 2^-24 (|x0| + |x1|), and the output's own
rounding for F16, 2^-11 |y| + 2^-25 (subnormals).  Angles: the F64 product of
position, scale and frequency, whose own roundings (4 * 2^-53 of the angle)
come on top.

Stored rows are compared with codes and scales computed in the definition's F32
steps, byte by byte; rotated ones are rotated by samhip_rope first, whose bits
the rotation on the way has.

Attention, as for samhip_prefix_attn: with keys and values as the blocks stand
for, operands of 22 bits and F32 sums, a score is off by at most
  ds = scale sum|q||k| (head_dim 2^-24 + 5 * 2^-22),
and |error| <= sum w|v| (2 ds + 2^-19 + (n / 16 + 48) 2^-24).  Weights times
value scales below 2^-16 of their query's largest are off by 2^-39 of it at
most (fp16's smallest step), on codes up to 128: + n 2^-32 max(w |d|)."""

import math

import numpy as np
import pytest

try:
    import torch
except ImportError:   # pragma: no cover
    torch = None

pytestmark = pytest.mark.gpu

DTYPES = {"f32": "float32", "f16": "float16"}


def dtype_of(name):
    return getattr(torch, DTYPES[name])


def describe(samhip, t):
    return samhip.tensor_nd(samhip.F16 if t.dtype == torch.float16 else samhip.F32, t.shape[::-1],
                            [v * t.element_size() for v in t.stride()[::-1]], t.data_ptr())


def strided(t, pad, dtype=None):
    held = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), device=t.device, dtype=dtype or t.dtype)
    held[:, :t.shape[1]] = t
    return held[:, :t.shape[1]]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# --- rotation -----------------------------------------------------------------


class Turn:
    """A rotation and its definition."""

    def __init__(self, hd, pairs, positions, halves=False, shared=False, theta=10000.0, scale=None):
        self.hd, self.pairs, self.positions, self.halves, self.shared, self.theta = hd, pairs, positions, halves, shared, theta
        self.scale = scale or [1.0] * len(pairs)

    def desc(self, samhip):
        return samhip.rope_desc(self.hd, self.pairs, self.positions.data_ptr(), samhip.ROPE_HALVES if self.halves else samhip.ROPE_ADJACENT,
                                samhip.ROPE_SHARED if self.shared else samhip.ROPE_AXIAL, self.theta, self.scale)

    def reference(self, x):
        """The rotation in F64, what F32 steps may be off by, and what angles may."""
        total = sum(self.pairs)
        x = x.double().view(x.shape[0], -1, self.hd)
        y, off = x.clone(), torch.zeros_like(x)
        p = 0
        for a, n in enumerate(self.pairs):
            for j in range(n):
                freq = self.theta ** (-p / total if self.shared else -j / n)
                angle = self.positions[:, a].double() * (self.scale[a] * freq)
                c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
                u, v = (p, p + total) if self.halves else (2 * p, 2 * p + 1)
                y[..., u], y[..., v] = x[..., u] * c - x[..., v] * s, x[..., u] * s + x[..., v] * c
                off[..., u] = off[..., v] = (x[..., u].abs() + x[..., v].abs()) * (4 * 2.0 ** -24 + 16 * 2.0 ** -53 * angle.abs()[:, None])
                p += 1
        return y.flatten(1), off.flatten(1)


ROPES = [
    # rows, heads, head_dim, pairs, halves, shared
    (1, 1, 2, [1], False, False),
    (1, 1, 64, [32], True, True),
    (7, 3, 6, [1, 1, 1], False, False),
    (33, 5, 32, [4, 6, 6], True, False),
    (201, 8, 32, [8, 8], False, False),
    (300, 2, 128, [16, 24, 24], True, True),
    (65, 3, 50, [3, 5], True, True),
    (19, 1, 256, [128], True, True),
    (40, 7, 96, [5, 1, 9], False, True),
    (1025, 4, 64, [7], True, False),
]


@pytest.mark.parametrize("case", range(len(ROPES)))
@pytest.mark.parametrize("types", ["f32 f32", "f32 f16", "f16 f32", "f16 f16"])
def test_rope(samhip, gpu_ctx, case, types):
    rows, heads, hd, pairs, halves, shared = ROPES[case]
    print("rope", ROPES[case], types, flush=True)
    xt, yt = types.split()
    for pad in (0, 3):
        g = torch.Generator(device="cuda").manual_seed(case)
        positions = torch.randint(-50, 5184, (rows, len(pairs)), device="cuda", generator=g, dtype=torch.int32)
        t = Turn(hd, pairs, positions, halves, shared)
        x = strided(torch.randn(rows, heads * hd, device="cuda", generator=g), pad, dtype_of(xt))
        held = torch.full((rows, heads * hd + pad), 7.0, device="cuda", dtype=dtype_of(yt))
        y = held[:, :heads * hd]
        want, off = t.reference(x)
        torch.cuda.synchronize()
        gpu_ctx.rope(t.desc(samhip), describe(samhip, x), describe(samhip, y))
        gpu_ctx.synchronize()
        if yt == "f16":
            off = off + want.abs() * 2.0 ** -11 + 2.0 ** -25
        assert ((y.double() - want).abs() <= off).all()
        assert (held[:, heads * hd:] == 7.0).all()
        if sum(pairs) * 2 < hd:   # values behind the pairs as they are
            tail = slice(2 * sum(pairs), hd)
            assert torch.equal(y.reshape(rows, heads, hd)[..., tail], x.reshape(rows, heads, hd)[..., tail].to(y.dtype))


@pytest.mark.parametrize("halves", [False, True])
def test_rope_in_place_far_positions_and_scales(samhip, gpu_ctx, halves):
    """Positions of the whole range, on a scale of a third: F64 angles to 2^30."""
    far = [2 ** 31 - 1, -2 ** 31, 123456789, -7, 0, 1]
    positions = ints([[far[i % 6], far[(i + 2) % 6]] for i in range(24)])
    t = Turn(64, [16, 16], positions, halves, theta=500000.0, scale=[1 / 3, -2.0])
    x = torch.randn(24, 3 * 64, device="cuda")
    want, off = t.reference(x)
    torch.cuda.synchronize()
    gpu_ctx.rope(t.desc(samhip), describe(samhip, x), describe(samhip, x))
    gpu_ctx.synchronize()
    assert ((x.double() - want).abs() <= off).all()


def test_rope_of_position_zero_and_non_finite_values(samhip, gpu_ctx):
    """Position 0 leaves every bit; an infinity or a NaN reaches its pair alone."""
    x = torch.randn(9, 4 * 32, device="cuda")
    t = Turn(32, [5, 11], ints([[0, 0]] * 9))
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    gpu_ctx.rope(t.desc(samhip), describe(samhip, x), describe(samhip, y))
    gpu_ctx.synchronize()
    assert torch.equal(x, y)
    for halves in (False, True):
        t = Turn(32, [4, 8], ints([[3, 5]] * 9), halves)
        x[2, 32 + 6], x[5, 64 + 30] = float("inf"), float("nan")   # a pair's, and one behind the pairs
        want, off = t.reference(torch.where(x.isfinite(), x, 0.0))
        torch.cuda.synchronize()
        gpu_ctx.rope(t.desc(samhip), describe(samhip, x), describe(samhip, y))
        gpu_ctx.synchronize()
        hit = torch.zeros_like(x, dtype=torch.bool)
        hit[2, 32 + 6] = hit[2, 32 + (18 if halves else 7)] = hit[5, 64 + 30] = True
        assert torch.equal(~y.isfinite(), hit)
        assert ((y.double() - want).abs() <= off)[~hit].all()


# --- what a block holds --------------------------------------------------------


def q8_0_blocks(x, x86):
    """d and codes of blocks x [..., 32] (numpy F32) in the definition's F32 steps."""
    amax = np.abs(x).max(-1, keepdims=True)
    d = (amax / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(amax > 0, np.float32(127) / amax if x86 else np.float32(1) / d, np.float32(0)).astype(np.float32)
    s = (x * inv).astype(np.float32)
    codes = np.rint(s) if x86 else np.trunc(s + np.copysign(np.float32(0.5), s).astype(np.float64))
    return d.astype(np.float16), codes.astype(np.int8)


def q4_0_blocks(x):
    first = np.abs(x).argmax(-1)[..., None]   # argmax: the first of equals
    d = (np.take_along_axis(x, first, -1) / np.float32(-8)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
    s = ((x * inv).astype(np.float32) + np.float32(8.5)).astype(np.float32)
    return d.astype(np.float16), np.minimum(np.trunc(s), 15).astype(np.uint8)


def packed(x, q4, x86=True):
    """Rows (F32 tensor) as cache bytes, a uint8 array [rows, row bytes]."""
    b = x.cpu().numpy().reshape(x.shape[0], -1, 32)
    d, c = q4_0_blocks(b) if q4 else q8_0_blocks(b, x86)
    if q4:
        c = c[..., :16] | (c[..., 16:] << 4)
    return np.concatenate([d.view(np.uint8), c.view(np.uint8)], -1).reshape(x.shape[0], -1)


def values(rows, q4):
    """Cache bytes (uint8 tensor [n, row bytes]) as F64 values [n, width]."""
    b = rows.reshape(rows.shape[0], rows.shape[1] // (18 if q4 else 34), -1)
    d = b[..., :2].contiguous().view(torch.float16).double()
    c = b[..., 2:]
    codes = torch.cat([c & 15, c >> 4], -1).double() - 8 if q4 else c.contiguous().view(torch.int8).double()
    return (d * codes).flatten(1)


class Pages:
    """Requests with n rows in the call and len positions, in pages dealt in no
    order; every cache byte nobody has is 0xff (NaN scales)."""

    def __init__(self, n, lens, kv_heads, hd, q4, page, seed=0, first=0, behind=0, byte_pad=0):
        self.n, self.lens, self.kv_heads, self.hd, self.q4, self.page = n, lens, kv_heads, hd, q4, page
        self.first, self.rows, self.width = first, first + sum(n) + behind, kv_heads * hd
        self.row_bytes = self.width // 32 * (18 if q4 else 34)
        counts = [-(-m // page) for m in lens]
        self.max_pages, self.total = max(1, max(counts)) + 1, sum(counts) + 2
        rng = np.random.default_rng(seed)
        order = rng.permutation(self.total)
        table = np.full((len(n), self.max_pages), -1, np.int32)
        for r, c in enumerate(counts):
            table[r, :c] = order[sum(counts[:r]):sum(counts[:r]) + c]
        self.table = table
        self.pages, self.len = ints(table.tolist()), ints(lens)
        self.starts = [first + sum(n[:r]) for r in range(len(n) + 1)]
        self.row_start = ints(self.starts)
        self.caches = [torch.full((self.total * page, self.row_bytes + byte_pad), 255, dtype=torch.uint8, device="cuda") for _ in "kv"]
        self.max_len = max(lens)

    def at(self, r, positions):
        p = np.asarray(positions)
        return torch.as_tensor(self.table[r][p // self.page].astype(np.int64) * self.page + p % self.page, device="cuda")

    def fill(self, seed=0, amp=1.0):
        """Positions 0 .. len - 1 of every request from N(0, 1) rows."""
        g = torch.Generator(device="cuda").manual_seed(seed)
        for r, m in enumerate(self.lens):
            if m:
                for i, c in enumerate(self.caches):
                    x = torch.randn(m, self.width, device="cuda", generator=g) * (amp if i == 0 else 1.0)
                    c[self.at(r, range(m)), :self.row_bytes] = torch.as_tensor(packed(x, self.q4), device="cuda")
        return self

    def desc(self, samhip):
        t = samhip.Q4_0 if self.q4 else samhip.Q8_0
        k, v = (samhip.tensor(t, self.width, c.shape[0], c.data_ptr(), nb1=c.stride(0)) for c in self.caches)
        return samhip.kv_cache(self.kv_heads, self.hd, self.page, k, v, len(self.n), self.max_pages, self.pages.data_ptr(), self.row_start.data_ptr(),
                               self.len.data_ptr())


# --- rows to and from a cache ---------------------------------------------------

STORES = [
    # rows, lengths, kv heads, head_dim, page
    ([1], [1], 1, 32, 1),
    ([1] * 9, [1, 2, 64, 65, 300, 7, 31, 32, 33], 4, 128, 16),
    ([5, 0, 33, 150, 1], [5, 9, 40, 150, 77], 3, 64, 41),
    ([700], [1000], 8, 32, 333),
    ([2, 3], [1, 2], 2, 32, 8),          # fewer positions than rows: the first have no place
    ([40], [200], 1, 64, 4096),
]


@pytest.mark.parametrize("case", range(len(STORES)))
@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("turned", [None, "halves", "adjacent", "odd halves"])
def test_write_and_read(samhip, gpu_ctx, case, q4, turned):
    n, lens, kv_heads, hd, page = STORES[case]
    print("write", STORES[case], "q4" if q4 else "q8", turned, flush=True)
    for pad in (0, 3):
        p = Pages(n, lens, kv_heads, hd, q4, page, seed=case, first=pad, behind=pad, byte_pad=2 * pad)
        g = torch.Generator(device="cuda").manual_seed(case)
        k, v = (strided(torch.randn(p.rows, p.width, device="cuda", generator=g), pad) for _ in "kv")
        rope, kt = None, k
        if turned:
            pairs = {"halves": [hd // 4, hd // 4], "adjacent": [hd // 8, hd // 8, hd // 8], "odd halves": [3, 7]}[turned]
            positions = torch.randint(0, 100000, (p.rows, len(pairs)), device="cuda", generator=g, dtype=torch.int32)
            turn = Turn(hd, pairs, positions, turned != "adjacent", turned == "halves")
            rope, kt = turn.desc(samhip), torch.empty(p.rows, p.width, device="cuda")
            torch.cuda.synchronize()
            gpu_ctx.rope(rope, describe(samhip, k), describe(samhip, kt))
        torch.cuda.synchronize()
        gpu_ctx.cache_write(p.desc(samhip), rope, describe(samhip, k), describe(samhip, v))
        gpu_ctx.synchronize()
        want = [torch.full_like(c, 255) for c in p.caches]
        read = [torch.full((p.rows, p.width), 7.0, device="cuda", dtype=torch.float64) for _ in "kv"]
        for i, x in enumerate((kt, v)):
            bytes_ = torch.as_tensor(packed(x, q4), device="cuda")
            for r, (rows, m) in enumerate(zip(n, lens)):
                s0, lost = p.starts[r], max(0, rows - m)
                read[i][s0:s0 + lost] = 0.0
                if rows > lost:
                    want[i][p.at(r, range(m - rows + lost, m)), :p.row_bytes] = bytes_[s0 + lost:s0 + rows]
                    read[i][s0 + lost:s0 + rows] = values(bytes_[s0 + lost:s0 + rows], q4)
        for i in range(2):
            assert torch.equal(p.caches[i], want[i])
        for out in ("f32", "f16"):
            held = [torch.full((p.rows, p.width + pad), 7.0, device="cuda", dtype=dtype_of(out)) for _ in "kv"]
            torch.cuda.synchronize()
            gpu_ctx.cache_read(p.desc(samhip), *(describe(samhip, h[:, :p.width]) for h in held))
            gpu_ctx.synchronize()
            for i in range(2):
                assert torch.equal(held[i][:, :p.width], read[i].to(dtype_of(out)))
                assert (held[i][:, p.width:] == 7.0).all()


@pytest.mark.parametrize("x86", [True, False])
def test_q8_0_rows_are_those_of_quantize_rows(samhip, x86):
    """Blocks of zeros, subnormals, one magnitude of both signs, ties and values
    whose scale overflows fp16, with a NaN and with an infinity."""
    rounding = samhip.ROUND_X86 if x86 else samhip.ROUND_REF
    with samhip.Context(0, samhip.COMPUTE_Q8_NATIVE, rounding) as ctx:
        rng = np.random.default_rng(5)
        x = rng.standard_normal((64, 64)).astype(np.float32)
        x[1] = 0
        x[2] *= 1e-42
        x[3, :32] = np.where(np.arange(32) % 2, -1.5, 1.5)
        x[4] = (np.arange(64) - 31.5) * 2
        x[4, 0] = -127
        x[5] *= 3e7
        x[6, 3] = np.nan
        x[7, 40] = np.inf
        x[8] *= 1e-30
        want = ctx.quantize(samhip.Q8_0, x, rounding)
        p = Pages([64], [64], 1, 64, False, 7)
        k = torch.as_tensor(x, device="cuda")
        torch.cuda.synchronize()
        ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, k))
        ctx.synchronize()
        at = p.at(0, range(64))
        for c in p.caches:
            assert np.array_equal(c[at].cpu().numpy(), want)
        out = [torch.empty_like(k) for _ in "kv"]
        ctx.cache_read(p.desc(samhip), *(describe(samhip, o) for o in out))
        ctx.synchronize()
        assert out[0][7, 32:].isnan().all() and out[0][7, :32].isfinite().all() and out[0][6].isfinite().all() and out[0][6, 3] == 0


def test_q4_0_edges(samhip, gpu_ctx):
    """Zeros, one magnitude of both signs (the first decides the scale's sign),
    a NaN (a zero), an infinity (its block reads NaN), scales that overflow."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((10, 32)).astype(np.float32)
    x[1] = 0
    x[2] = np.where(np.arange(32) % 2, 2.0, -2.0)
    x[3] = -x[2]
    x[4, 5] = np.nan
    x[5, 6] = -np.inf
    x[6] *= 1e-42
    x[7] *= 3e6
    clean = np.where(np.isnan(x), 0, x).astype(np.float32)
    p = Pages([10], [10], 1, 32, True, 3)
    k = torch.as_tensor(x, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, k))
    out = [torch.empty_like(k) for _ in "kv"]
    gpu_ctx.cache_read(p.desc(samhip), *(describe(samhip, o) for o in out))
    gpu_ctx.synchronize()
    keep = [0, 1, 2, 3, 4, 8, 9]
    with np.errstate(over="ignore", invalid="ignore"):
        want = packed(torch.as_tensor(clean[keep]), True)
    assert np.array_equal(p.caches[0][p.at(0, keep)].cpu().numpy(), want)
    assert out[1][5].isnan().all() and (out[0][6] == 0).all() and not out[0][7].isfinite().all()
    # the first value's sign has code 0, -8 steps; the other's 15, 7 of them
    assert out[0][2].tolist() == [-2.0, 1.75] * 16 and out[0][3].tolist() == [2.0, -1.75] * 16 and out[0][4, 5] == 0


def test_rows_and_pages_that_do_not_exist(samhip, gpu_ctx):
    """Page numbers outside the cache, lengths beyond the table and row tables
    beyond the rows: nothing outside is touched, what is there is served."""
    p = Pages([4, 4, 4], [8, 8, 8], 1, 32, True, 4)
    table = p.table.copy()
    free = [i for i in range(p.total) if i != table[0, 0]]   # no page has two owners
    table[0, 1], table[1, 0], table[1, 1], table[2, :] = p.total, -5, 2 ** 31 - 1, [free[0], free[1], 2 ** 30]
    p.pages.copy_(ints(table.tolist()))
    p.len.copy_(ints([8, 8, 2 ** 31 - 1]))
    p.row_start.copy_(ints([-9, 4, 8, 2 ** 31 - 1]))
    k = torch.randn(12, 32, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, k))
    out = [torch.full_like(k, 7.0) for _ in "kv"]
    gpu_ctx.cache_read(p.desc(samhip), *(describe(samhip, o) for o in out))
    gpu_ctx.synchronize()
    assert all((c == 255).all() for c in p.caches) and all((o == 0).all() for o in out)
    p.len.copy_(ints([4, -1, 6]))
    torch.cuda.synchronize()
    gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, k))
    gpu_ctx.cache_read(p.desc(samhip), *(describe(samhip, o) for o in out))
    gpu_ctx.synchronize()
    want = values(torch.as_tensor(packed(k, True), device="cuda"), True)
    want[4:8] = 0
    for o in out:
        assert torch.equal(o.double(), want)


# --- attention ------------------------------------------------------------------


class Attend:
    def __init__(self, pages, heads, causal=False, pad=0, seed=0, amp=1.0, scale=None):
        self.p, self.heads, self.causal = pages, heads, causal
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q = strided(torch.randn(pages.rows, heads * pages.hd, device="cuda", generator=g) * amp, pad)
        self.scale = pages.hd ** -0.5 if scale is None else scale
        self.held = torch.full((pages.rows, heads * pages.hd + pad), 7.0, device="cuda")
        self.out = self.held[:, :heads * pages.hd]
        self.max_len = pages.max_len

    def desc(self, samhip):
        return samhip.cache_attn_desc(self.heads, self.scale, self.p.desc(samhip), describe(samhip, self.q), describe(samhip, self.out), self.max_len,
                                      self.causal)

    def reference(self, lens=None, n=None, starts=None):
        p, h, hd, group = self.p, self.heads, self.p.hd, self.heads // self.p.kv_heads
        lens, n, starts = lens or p.lens, n or p.n, starts or p.starts
        ref = torch.full((p.rows, h * hd), 7.0, device="cuda", dtype=torch.float64)
        bound = torch.zeros_like(ref)
        for r, rows in enumerate(n):
            if not rows:
                continue
            m, s0 = min(lens[r], self.max_len), starts[r]
            q = self.q[s0:s0 + rows].double().view(rows, h, hd)
            if not m:
                ref[s0:s0 + rows] = 0.0
                continue
            at = p.at(r, range(m))
            k, v = (values(c[at][:, :p.row_bytes], p.q4).view(m, p.kv_heads, hd) for c in p.caches)
            seen = torch.ones(rows, m, dtype=torch.bool, device="cuda")
            if self.causal:
                seen = torch.arange(m, device="cuda")[None, :] <= torch.arange(rows, device="cuda")[:, None] + (lens[r] - rows)
            most_d = v.view(m, -1, 32).abs().amax(-1).view(m, p.kv_heads, -1).amax(-1) / (8 if p.q4 else 127)
            for head in range(h):
                kk, vv = k[:, head // group], v[:, head // group]
                s = (q[:, head] @ kk.t()) * self.scale
                mag = (q[:, head].abs() @ kk.abs().t()) * abs(self.scale)
                some = seen.any(1, keepdim=True)
                top = s.masked_fill(~seen, -torch.inf).amax(1, keepdim=True)
                w = torch.where(seen, torch.exp(s - torch.where(some, top, 0.0)), 0.0)
                w = w / torch.where(some, w.sum(1, keepdim=True), 1.0)
                cols = slice(head * hd, (head + 1) * hd)
                ref[s0:s0 + rows, cols] = w @ vv
                ds = mag.masked_fill(~seen, 0.0).amax(1, keepdim=True) * (hd * 2.0 ** -24 + 5 * 2.0 ** -22)
                bound[s0:s0 + rows, cols] = (w @ vv.abs()) * (2 * ds + 2.0 ** -19 + (m / 16 + 48) * 2.0 ** -24) + \
                    m * 2.0 ** -32 * (w * most_d[:, head // group]).amax(1, keepdim=True)
        return ref, bound

    def run(self, samhip, ctx):
        torch.cuda.synchronize()
        ctx.cache_attn(self.desc(samhip))
        ctx.synchronize()

    def check(self, samhip, ctx):
        ref, bound = self.reference()
        self.run(samhip, ctx)
        self.verify(ref, bound)

    def verify(self, ref, bound):
        err = (self.out.double() - ref).abs()
        assert (err <= bound).all(), (err / bound.clamp(min=1e-30)).max().item()
        assert (self.held[:, self.heads * self.p.hd:] == 7.0).all()


ATTENDS = [
    # rows, lengths, heads, kv heads, page
    ([1], [0], 1, 1, 16),
    ([1], [1], 2, 1, 16),
    ([1] * 8, [5184, 64, 1, 33, 2, 0, 31, 32], 8, 8, 64),
    ([1] * 70, [(37 * i) % 700 for i in range(70)], 8, 2, 41),
    ([5, 0, 150, 31, 0, 1, 64], [9, 3, 300, 1031, 0, 77, 64], 12, 4, 41),
    ([3, 40], [0, 50], 4, 4, 7),
    ([2, 3], [700, 20], 16, 1, 1),
    ([9] * 5, [700, 1, 256, 257, 0], 3, 3, 256),
    ([4, 1], [3000, 129], 24, 2, 333),
    ([300], [300], 2, 2, 128),
]


@pytest.mark.parametrize("case", range(len(ATTENDS)))
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("q4", [False, True])
def test_cache_attn(samhip, gpu_ctx, case, hd, q4):
    n, lens, heads, kv_heads, page = ATTENDS[case]
    print("cache_attn", ATTENDS[case], hd, "q4" if q4 else "q8", flush=True)
    for causal in (False, True):
        p = Pages(n, lens, kv_heads, hd, q4, page, seed=case, first=(0, 2)[causal], behind=(0, 3)[causal], byte_pad=(0, 6)[causal]).fill(case)
        Attend(p, heads, causal, pad=(0, 3)[causal], seed=case).check(samhip, gpu_ctx)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("q4", [False, True])
def test_peaked_scores(samhip, gpu_ctx, q4, rows):
    """Scores of hundreds: one key takes all the weight, the largest so far moves."""
    p = Pages([rows, rows], [2000, 265], 2, 64, q4, 64, seed=3).fill(3, amp=6.0)
    Attend(p, 4, True, amp=6.0, seed=3).check(samhip, gpu_ctx)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("scale", [0.0, -0.125, -2.0, 1e-30])
def test_scales_of_either_sign_and_zero(samhip, gpu_ctx, scale, rows):
    p = Pages([rows, rows], [700, 65], 2, 64, True, 64, seed=4).fill(4)
    Attend(p, 4, True, seed=4, scale=scale).check(samhip, gpu_ctx)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("exponent", [-100, -40, 40, 100])
def test_queries_of_any_magnitude(samhip, gpu_ctx, exponent, rows):
    p = Pages([rows], [700], 2, 64, False, 64, seed=5).fill(5)
    a = Attend(p, 4, seed=5, scale=0.125 * 2.0 ** -exponent if abs(exponent) < 100 else 2.0 ** -math.copysign(100, exponent))
    a.q.mul_(2.0 ** exponent)
    a.q[0, :64] = 0.0
    a.check(samhip, gpu_ctx)


def scale_blocks(p, r, which, positions, factor, block=None):
    """Multiplies the scales of a request's blocks (which: 0 keys, 1 values)."""
    c, at = p.caches[which], p.at(r, positions)
    rows = c[at]
    b = rows[:, :p.row_bytes].reshape(len(at), -1, 18 if p.q4 else 34)
    d = b[..., :2].contiguous().view(torch.float16).float() * factor
    new = d.half().view(torch.uint8)
    if block is None:
        b[..., :2] = new
    else:
        b[:, block, :2] = new[:, block]
    rows[:, :p.row_bytes] = b.reshape(len(at), -1)
    c[at] = rows


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("q4", [False, True])
def test_values_of_many_magnitudes(samhip, gpu_ctx, q4, rows):
    """Value rows of zeros, of 2^-12 and 2^14 times the others, in runs and alone."""
    p = Pages([rows, rows], [900, 700], 2, 64, q4, 64, seed=6).fill(6)
    scale_blocks(p, 0, 1, range(0, 128), 0.0)
    scale_blocks(p, 0, 1, range(200, 300), 2.0 ** -12)
    scale_blocks(p, 0, 1, range(400, 432), 2.0 ** 14)
    scale_blocks(p, 1, 1, [5, 77, 300], 2.0 ** 14)
    scale_blocks(p, 1, 1, range(600, 700), 2.0 ** -13)
    Attend(p, 4, True, seed=6).check(samhip, gpu_ctx)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("below", [10.0, 18.5])
def test_large_values_of_little_weight(samhip, gpu_ctx, below, rows):
    """The second half's values are 2^20 times the first's, at scores `below`
    nats under them: both count."""
    p = Pages([rows], [512], 1, 32, True, 64, seed=7).fill(7)
    a = Attend(p, 1, seed=7, scale=1.0)
    a.q.fill_(1.0)
    k = torch.zeros(512, 32, device="cuda")
    k[256:] = -below / 32
    p.caches[0][p.at(0, range(512))] = torch.as_tensor(packed(k, True), device="cuda")
    scale_blocks(p, 0, 1, range(0, 256), 2.0 ** -9)
    scale_blocks(p, 0, 1, range(256, 512), 2.0 ** 11)
    a.check(samhip, gpu_ctx)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("q4", [False, True])
def test_non_finite_blocks_reach_only_queries_that_see_them(samhip, gpu_ctx, q4, rows):
    """Key 690 of request 0 has a NaN scale in kv head 0; value 695 an infinite
    one in kv head 1's second block."""
    p = Pages([rows, 3], [700, 40], 2, 64, q4, 41, seed=8).fill(8)
    a = Attend(p, 4, True, seed=8)
    ref, bound = a.reference()
    scale_blocks(p, 0, 0, [690], float("nan"), 1)
    scale_blocks(p, 0, 1, [695], float("inf"), 3)
    a.run(samhip, gpu_ctx)
    hit = torch.zeros(rows + 3, 4, 64, dtype=torch.bool, device="cuda")
    for i in range(rows):
        position = 700 - rows + i
        hit[i, :2] |= position >= 690
        hit[i, 2:, 32:] |= position >= 695
    out = a.out.view(-1, 4, 64)
    assert torch.equal(~out.isfinite(), hit)
    err, most = (out.double() - ref.view(-1, 4, 64)).abs(), bound.view(-1, 4, 64)
    assert (err[~hit] <= most[~hit]).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_and_lengths_that_do_not_exist(samhip, gpu_ctx, rows):
    """A page outside the cache hides its positions; lengths are cut to max_len,
    the table and zero; rows outside the row table are left alone."""
    p = Pages([rows] * 3, [300, 300, 300], 2, 64, True, 41, seed=9).fill(9)
    a = Attend(p, 4, seed=9)
    table = p.table.copy()
    table[1, 2] = p.total
    table[2, 0] = -7
    p.pages.copy_(ints(table.tolist()))
    p.len.copy_(ints([2 ** 31 - 1, 300, 200]))
    p.row_start.copy_(ints([-3, rows, 2 * rows, 2 ** 31 - 1]))
    a.max_len = 290
    a.run(samhip, gpu_ctx)
    keys = [range(290), [i for i in range(290) if i // 41 != 2], range(41, 200)]
    q = a.q.double().view(-1, 4, 64)
    for r in range(3):
        at = p.at(r, keys[r])
        k, v = (values(c[at][:, :p.row_bytes], True).view(-1, 2, 64) for c in p.caches)
        for h in range(4):
            w = torch.softmax(q[r * rows:(r + 1) * rows, h] @ k[:, h // 2].t() * a.scale, -1)
            got = a.out.view(-1, 4, 64)[r * rows:(r + 1) * rows, h].double()
            assert ((got - w @ v[:, h // 2]).abs() <= 1e-5).all()
    p.len.copy_(ints([0, -4, 0]))
    a.run(samhip, gpu_ctx)
    assert (a.out == 0).all()


def test_captured_replays_follow_the_tables(samhip, gpu_ctx):
    """One graph of a step (rotated queries, rows written, attention), replayed
    as the requests' caches grow; each replay gives the eager step's bits."""
    n, steps = 6, 4
    p = Pages([1] * n, [20 + 40 * i + steps for i in range(n)], 2, 64, True, 16, seed=11).fill(11)
    a = Attend(p, 4, True, seed=11)
    k, v, q = (torch.zeros(n, w, device="cuda") for w in (128, 128, 256))
    positions = torch.zeros(n, 1, device="cuda", dtype=torch.int32)
    turn = Turn(64, [32], positions, True, True)

    def step():
        gpu_ctx.rope(turn.desc(samhip), describe(samhip, q), describe(samhip, a.q))
        gpu_ctx.cache_write(p.desc(samhip), turn.desc(samhip), describe(samhip, k), describe(samhip, v))
        gpu_ctx.cache_attn(a.desc(samhip))

    torch.cuda.synchronize()
    step()   # staging
    gpu_ctx.capture_begin()
    step()
    graph = gpu_ctx.capture_end()
    fresh = [c.clone() for c in p.caches]
    rolls = []
    for replayed in (False, True):
        g = torch.Generator(device="cuda").manual_seed(1)
        for c, f in zip(p.caches, fresh):
            c.copy_(f)
        outs = []
        for t in range(steps):
            for x in (k, v, q):
                x.normal_(generator=g)
            lens = [20 + 40 * i + t + 1 for i in range(n)]
            p.len.copy_(ints(lens))
            positions.copy_(ints([[m - 1] for m in lens]))
            a.held.fill_(7.0)
            torch.cuda.synchronize()
            if replayed:
                graph.launch()
            else:
                step()
            gpu_ctx.synchronize()
            outs.append((a.out.clone(), *[c.clone() for c in p.caches]))
            ref, bound = a.reference(lens)
            a.verify(ref, bound)
            torch.randn(512, 256, device="cuda") @ torch.randn(256, 64, device="cuda")
        rolls.append(outs)
    graph.destroy()
    for e, r in zip(*rolls):
        for x, y in zip(e, r):
            assert torch.equal(x, y)


def test_a_service_on_its_own_stream(samhip):
    """Prompts and then single tokens, all on a caller's stream and with other
    work queued before: rows stored step by step serve as those stored at once."""
    with samhip.Context(0) as ctx:
        lens, hd, kv, heads = [40, 7, 129], 32, 4, 8
        g = torch.Generator(device="cuda").manual_seed(12)
        total = sum(lens)
        rows = {n: torch.randn(total, w * hd, device="cuda", generator=g) for n, w in (("q", heads), ("k", kv), ("v", kv))}
        grid = torch.stack([torch.arange(total, device="cuda") // 9, torch.arange(total, device="cuda") % 9], 1).int()
        turn = lambda positions: Turn(hd, [8, 8], positions)  # noqa: E731
        stream = torch.cuda.Stream()
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            def serve(p, picks):
                """The call of rows `picks` (of all), p.n to a request."""
                x = {n: t[picks].contiguous() for n, t in rows.items()}
                at = grid[picks].contiguous()
                ctx.rope(turn(at).desc(samhip), describe(samhip, x["q"]), describe(samhip, x["q"]))
                ctx.cache_write(p.desc(samhip), turn(at).desc(samhip), describe(samhip, x["k"]), describe(samhip, x["v"]))
                out = torch.empty_like(x["q"])
                ctx.cache_attn(samhip.cache_attn_desc(heads, hd ** -0.5, p.desc(samhip), describe(samhip, x["q"]), describe(samhip, out), max(lens), True))
                keep.append((x, at, p))
                return out

            keep, starts = [], [sum(lens[:r]) for r in range(3)]
            big = torch.randn(2048, 2048, device="cuda")
            for _ in range(4):
                big = big @ big * 1e-3
            p = Pages(lens, lens, kv, hd, True, 16, seed=12)
            once = serve(p, list(range(total)))
            bytes_once = [c.clone() for c in p.caches]
            for c in p.caches:
                c.fill_(255)
            # all but the last 3 of each as prompts, then one by one
            split = Pages([m - 3 for m in lens], [m - 3 for m in lens], kv, hd, True, 16, seed=12)
            split.pages, split.caches, split.max_pages = p.pages, p.caches, p.max_pages
            picks = [s + i for s, m in zip(starts, lens) for i in range(m - 3)]
            got = torch.empty_like(once)
            got[picks] = serve(split, picks)
            for t in (3, 2, 1):
                one = Pages([1] * 3, [m - t + 1 for m in lens], kv, hd, True, 16, seed=12)
                one.pages, one.caches, one.max_pages = p.pages, p.caches, p.max_pages
                picks = [s + m - t for s, m in zip(starts, lens)]
                got[picks] = serve(one, picks)
                keep.append(one)
        stream.synchronize()
        for c, b in zip(p.caches, bytes_once):
            assert torch.equal(c, b)
        # weights and sums in another order: the tolerance of two results of one definition
        assert ((got - once).abs() <= 2 * 2.0 ** -17 * once.abs().amax()).all()
        ctx.set_stream(None)


# --- large, many, at once ----------------------------------------------------------


@pytest.mark.parametrize("rows,requests,longest", [([1, 0, 2], 300, 400), ([1], 5000, 300), ([1], 1500, 60), ([40], 80, 300)])
def test_many_requests(samhip, gpu_ctx, rows, requests, longest):
    """More requests than a wave's lanes, rows of some and of none; lengths that
    leave one part of keys, and several."""
    print("many", rows, requests, longest, flush=True)
    n = [rows[i % len(rows)] for i in range(requests)]
    lens = [max(n[i], 137 * i % longest) for i in range(requests)]
    lens[-3] = 8 * longest   # one of many parts
    p = Pages(n, lens, 2, 32, True, 16, seed=13, first=2, behind=3)
    for i, c in enumerate(p.caches):   # all positions at once
        at = torch.cat([p.at(r, range(m)) for r, m in enumerate(lens)])
        g = torch.Generator(device="cuda").manual_seed(i)
        c[at, :p.row_bytes] = torch.as_tensor(packed(torch.randn(len(at), 64, device="cuda", generator=g), True), device="cuda")
    Attend(p, 4, True, seed=13).check(samhip, gpu_ctx)
    # the same tables for rows to and from the cache
    k = torch.randn(p.rows, 64, device="cuda")
    out = [torch.full_like(k, 7.0) for _ in "kv"]
    torch.cuda.synchronize()
    gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, k))
    gpu_ctx.cache_read(p.desc(samhip), *(describe(samhip, o) for o in out))
    gpu_ctx.synchronize()
    want = torch.full_like(k, 7.0)
    here = slice(p.starts[0], p.starts[-1])
    want[here] = values(torch.as_tensor(packed(k[here], True), device="cuda"), True).float()
    for i in range(2):
        assert torch.equal(out[i], want)
        at = torch.cat([p.at(r, range(m - a, m)) for r, (a, m) in enumerate(zip(n, lens)) if a])
        assert torch.equal(values(p.caches[i][at][:, :p.row_bytes], True).float(), want[here])


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("hd,group", [(32, 24), (64, 12), (128, 6), (128, 8), (64, 3)])
def test_places_of_two_operands_and_fewer(samhip, gpu_ctx, q4, hd, group):
    """Single rows of groups of heads between a whole operand's places and two's."""
    p = Pages([1, 1, 0, 1], [3001, 40, 5, 700], 2, hd, q4, 32, seed=14).fill(14)
    Attend(p, 2 * group, True, seed=14).check(samhip, gpu_ctx)


def test_as_many_kv_heads_as_there_may_be(samhip, gpu_ctx):
    p = Pages([1, 1], [3, 600], 1024, 32, True, 64, seed=15).fill(15)
    Attend(p, 1024, seed=15).check(samhip, gpu_ctx)
    p = Pages([1], [5], 4096, 32, False, 4, seed=16).fill(16)
    Attend(p, 4096, seed=16).check(samhip, gpu_ctx)


@pytest.mark.parametrize("stride,rows,lens", [(2 ** 26 + 2, 1, [33, 40]), (2 ** 26 + 4, 20, [33, 40]), (2 ** 23, 1, [600])])
def test_offsets_past_32_bits(samhip, gpu_ctx, stride, rows, lens):
    """Caches of more than 4 GiB: rows a long way from each other."""
    print("offsets", stride, rows, lens, flush=True)
    row_bytes = 4 * 64 // 32 * 18
    p = Pages([rows] * len(lens), lens, 4, 64, True, 16, seed=17, byte_pad=stride - row_bytes)
    assert p.caches[0].numel() > 2 ** 32

    def rows_of(c, at):
        return c[:, :p.row_bytes][at]

    k, v = (torch.randn(p.rows, 256, device="cuda") for _ in "kv")
    for i, c in enumerate(p.caches):
        narrow = c[:, :p.row_bytes]
        for r, m in enumerate(lens):
            g = torch.Generator(device="cuda").manual_seed(10 * r + i)
            narrow[p.at(r, range(m))] = torch.as_tensor(packed(torch.randn(m, 256, device="cuda", generator=g), True), device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, v))
    out = [torch.empty_like(k) for _ in "kv"]
    gpu_ctx.cache_read(p.desc(samhip), *(describe(samhip, o) for o in out))
    gpu_ctx.synchronize()
    for x, o, c in zip((k, v), out, p.caches):
        bytes_ = torch.as_tensor(packed(x, True), device="cuda")
        assert torch.equal(o.double(), values(bytes_, True))
        for r, m in enumerate(lens):
            assert torch.equal(rows_of(c, p.at(r, range(m - rows, m))), bytes_[r * rows:(r + 1) * rows])
    a = Attend(p, 4, True, seed=17)
    near = Pages([rows] * len(lens), lens, 4, 64, True, 16, seed=17)   # the same rows next to each other, for the reference
    for c, f in zip(near.caches, p.caches):
        for r, m in enumerate(lens):
            c[near.at(r, range(m))] = rows_of(f, p.at(r, range(m)))
    b = Attend(near, 4, True, seed=17)
    ref, bound = b.reference()
    a.run(samhip, gpu_ctx)
    a.verify(ref, bound)


@pytest.mark.parametrize("rows", [1, 40])
def test_caches_without_pages(samhip, gpu_ctx, rows):
    """Pages larger than the cache, and requests without any: zeros, and nothing
    written."""
    for page, max_pages in ((1 << 20, 3), (16, 0)):
        p = Pages([rows] * 2, [50, 40], 2, 32, False, 16, seed=18).fill(18)
        p.page, p.max_pages = page, max_pages
        before = [c.clone() for c in p.caches]
        k = torch.randn(p.rows, 64, device="cuda")
        out = [torch.full_like(k, 7.0) for _ in "kv"]
        a = Attend(p, 2, seed=18)
        torch.cuda.synchronize()
        gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, k))
        gpu_ctx.cache_read(p.desc(samhip), *(describe(samhip, o) for o in out))
        a.run(samhip, gpu_ctx)
        assert (a.out == 0).all() and all((o == 0).all() for o in out)
        assert all(torch.equal(c, b) for c, b in zip(p.caches, before))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_queries_that_are_not_finite_spoil_their_head_alone(samhip, gpu_ctx, rows, bad):
    p = Pages([rows, rows], [700, 33], 2, 64, True, 64, seed=19).fill(19)
    a = Attend(p, 4, seed=19)
    ref, bound = a.reference()
    a.q[0, 64 + 5] = bad
    a.q[rows, 3 * 64 + 40] = -bad
    a.run(samhip, gpu_ctx)
    hit = torch.zeros(2 * rows, 4, 64, dtype=torch.bool, device="cuda")
    hit[0, 1] = hit[rows, 3] = True
    out = a.out.view(-1, 4, 64)
    assert torch.equal(~out.isfinite(), hit)
    assert ((out.double() - ref.view(-1, 4, 64)).abs() <= bound.view(-1, 4, 64))[~hit].all()


def test_two_contexts_at_once(samhip):
    """Calls of two contexts, neither waiting for the other: scratch is each one's own."""
    with samhip.Context(0) as one, samhip.Context(0) as two:
        work = []
        for i, ctx in enumerate((one, two)):
            p = Pages([1] * (5 + 70 * i), [900 - 11 * j for j in range(5 + 70 * i)], 2, 64, True, 16, seed=20 + i).fill(20 + i)
            a = Attend(p, 4, True, seed=20 + i)
            work.append((ctx, a, a.reference()))
        torch.cuda.synchronize()
        for _ in range(20):
            for ctx, a, _ in work:
                ctx.cache_attn(a.desc(samhip))
        for ctx, a, (ref, bound) in work:
            ctx.synchronize()
            a.verify(ref, bound)


def test_two_graphs_that_share_scratch(samhip, gpu_ctx):
    """Graphs of few and of many requests, replayed in turn with eager work between."""
    work = []
    for i, (n, lens) in enumerate((([1] * 3, [2000, 5, 800]), ([1] * 90, [700 - 7 * j for j in range(90)]), ([40] * 3, [900, 41, 300]))):
        p = Pages(n, lens, 2, 64, i == 1, 16, seed=30 + i).fill(30 + i)
        a = Attend(p, 4, True, seed=30 + i)
        ref, bound = a.reference()
        a.run(samhip, gpu_ctx)   # scratch
        a.verify(ref, bound)
        work.append([a, ref, bound, a.out.clone()])
    graphs = []
    for a, *_ in work:
        gpu_ctx.capture_begin()
        gpu_ctx.cache_attn(a.desc(samhip))
        graphs.append(gpu_ctx.capture_end())
    for turn in range(4):
        for (a, ref, bound, eager), graph in zip(work, graphs):
            a.held.fill_(7.0)
            torch.cuda.synchronize()
            graph.launch()
            gpu_ctx.synchronize()
            assert torch.equal(a.out, eager)
            torch.randn(256, 256, device="cuda") @ torch.randn(256, 64, device="cuda")
        work[turn % 3][0].run(samhip, gpu_ctx)
    for graph in graphs:
        graph.destroy()


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kv_heads", [2, 4, 6, 8])
def test_waves_with_heads_of_their_own(samhip, gpu_ctx, kv_heads, hd, q4):
    """Enough requests of single rows that a workgroup takes two or four kv heads;
    lengths that leave waves without keys."""
    lens = [(53 * i + 1) % 977 for i in range(48)]
    p = Pages([1] * 48, lens, kv_heads, hd, q4, 41, seed=40, behind=2).fill(40)
    Attend(p, 2 * kv_heads, True, seed=40).check(samhip, gpu_ctx)
    scale_blocks(p, 20, 1, [lens[20] - 1], float("inf"), kv_heads * hd // 32 - 1)   # of the last kv head's last block
    a = Attend(p, 2 * kv_heads, seed=40)
    a.run(samhip, gpu_ctx)
    hit = torch.zeros(48, 2 * kv_heads, hd, dtype=torch.bool, device="cuda")
    hit[20, -2:, -32:] = True
    assert torch.equal(~a.out[:48].view(48, 2 * kv_heads, hd).isfinite(), hit)


@pytest.mark.parametrize("rows", [1, 40])
def test_scales_near_the_largest_number(samhip, gpu_ctx, rows):
    """Scores of ordinary size from subnormal queries: no product on the way overflows."""
    p = Pages([rows, rows], [700, 65], 2, 64, False, 64, seed=41).fill(41)
    a = Attend(p, 4, seed=41, scale=3.3e38)
    a.q.mul_(2.0 ** -128)
    a.check(samhip, gpu_ctx)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows", [4, 8, 9, 16, 32, 33])
def test_several_tiles_of_few_places(samhip, gpu_ctx, rows, hd, q4):
    """Requests whose places fill whole tiles of the form for few, one more, and those on either side of the other form."""
    p = Pages([rows, rows - 1, rows], [1300, rows, 333], 4, hd, q4, 16, seed=42, first=1, behind=1).fill(42)
    for causal in (False, True):
        Attend(p, 4, causal, pad=3, seed=42).check(samhip, gpu_ctx)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("rows", [24, 25, 70, 129])
def test_tiles_of_32_keys_of_head_dim_128(samhip, gpu_ctx, rows, q4):
    """Lengths on either side of the many-place form's tiles and parts."""
    for lens in ([64, 65, 33], [2000, 31, 97]):
        p = Pages([rows, 3, rows], lens, 2, 128, q4, 41, seed=43, behind=1).fill(43)
        for causal in (False, True):
            Attend(p, 2, causal, seed=43).check(samhip, gpu_ctx)


# --- value scales of one tile that lie far apart ------------------------------------


def tight(a):
    """The definition in F64 of every row of an Attend, and what it may be off by,
    key by key: a weight is off by its score's error ds (as above, of its own key)
    and, through the sum of weights, by their mean; then the operands' and sums'
    roundings, and fp16's half step 2^-25 of each product, of which the largest is
    2^13 at least: 2^-38 of it on codes up to 128."""
    p, hd, group = a.p, a.p.hd, a.heads // a.p.kv_heads
    ref = torch.full((p.rows, a.heads * hd), 7.0, device="cuda", dtype=torch.float64)
    bound = torch.zeros_like(ref)
    for r, (n, m) in enumerate(zip(p.n, p.lens)):
        if not n or not m:
            continue
        s0 = p.starts[r]
        q = a.q[s0:s0 + n].double().view(n, a.heads, hd)
        at = p.at(r, range(m))
        k, v = (values(c[at][:, :p.row_bytes], p.q4).view(m, p.kv_heads, hd) for c in p.caches)
        block = 18 if p.q4 else 34
        d = p.caches[1][at][:, :p.row_bytes].reshape(m, -1, block)[..., :2].contiguous().view(torch.float16).double().abs()
        d = d.view(m, p.kv_heads, -1).amax(-1)
        hidden = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        if a.causal:
            hidden = torch.arange(m, device="cuda")[None, :] > torch.arange(n, device="cuda")[:, None] + (m - n)
        for h in range(a.heads):
            kk, vv, dd = k[:, h // group], v[:, h // group], d[:, h // group]
            w = torch.softmax(((q[:, h] @ kk.t()) * a.scale).masked_fill(hidden, -torch.inf), -1)
            ds = (q[:, h].abs() @ kk.abs().t()) * abs(a.scale) * (hd * 2.0 ** -24 + 5 * 2.0 ** -22)
            off = ds + (w * ds).sum(-1, keepdim=True) + 2.0 ** -19 + (m / 16 + 48) * 2.0 ** -24
            cols = slice(h * hd, (h + 1) * hd)
            ref[s0:s0 + n, cols] = w @ vv
            bound[s0:s0 + n, cols] = 1.01 * (w * off) @ vv.abs() + m * 2.0 ** -31 * (w * dd).amax(1, keepdim=True)
    return ref, bound


def small_and_large(q4):
    """Factors that bring value scales of N(0, 1) to about 2^-14.4, and those 2^29 times as large."""
    return (2.0 ** -13, 2.0 ** 16) if q4 else (2.0 ** -9, 2.0 ** 20)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("from_the_end", [1, 2, 20])
def test_large_value_scales_that_some_queries_do_not_see(samhip, gpu_ctx, from_the_end, rows, hd, q4):
    """One value row 2^29 times the others inside a tile, hidden from the first
    rows: those have the bits that they have with an ordinary one there, and the
    accuracy that they have without it."""
    if from_the_end >= rows:
        pytest.skip("seen by all")
    print("hidden scale", from_the_end, rows, hd, q4, flush=True)
    small, large = small_and_large(q4)
    outs, m = [], 702
    for factor in (small, large):
        p = Pages([rows, rows], [m, 300], 2, hd, q4, 41, seed=50).fill(50)
        scale_blocks(p, 0, 1, range(m), small)
        scale_blocks(p, 0, 1, [m - from_the_end], factor / small)
        a = Attend(p, 4, True, seed=50)
        ref, bound = tight(a)
        a.run(samhip, gpu_ctx)
        a.verify(ref, bound)
        outs.append(a.out[:rows - from_the_end].clone())
    assert torch.equal(*outs)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("place", [5, 250, 511])
def test_large_value_scales_of_no_weight(samhip, gpu_ctx, place, rows, hd, q4):
    """One value row 2^29 times the others, whose key is 80 nats below theirs: in
    the first tile, inside one, and last."""
    print("weightless scale", place, rows, hd, q4, flush=True)
    small, large = small_and_large(q4)
    p = Pages([rows], [512], 1, hd, q4, 64, seed=51).fill(51)
    k = torch.zeros(512, hd, device="cuda")
    k[place] = -80 / hd
    p.caches[0][p.at(0, range(512))] = torch.as_tensor(packed(k, q4), device="cuda")
    scale_blocks(p, 0, 1, range(512), small)
    scale_blocks(p, 0, 1, [place], large / small)
    a = Attend(p, 2, seed=51, scale=1.0)
    a.q.fill_(1.0)
    ref, bound = tight(a)
    a.run(samhip, gpu_ctx)
    a.verify(ref, bound)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("below", [10.0, 18.5, 30.0])
@pytest.mark.parametrize("place", [250, 275])
def test_value_scales_that_change_inside_a_tile(samhip, gpu_ctx, place, below, rows, hd):
    """As test_large_values_of_little_weight, 2^29 apart and the change on no tile's border."""
    p = Pages([rows], [512], 1, hd, True, 64, seed=52).fill(52)
    k = torch.zeros(512, hd, device="cuda")
    k[place:] = -below / hd
    p.caches[0][p.at(0, range(512))] = torch.as_tensor(packed(k, True), device="cuda")
    small, large = small_and_large(True)
    scale_blocks(p, 0, 1, range(0, place), small)
    scale_blocks(p, 0, 1, range(place, 512), large)
    a = Attend(p, 1, seed=52, scale=1.0)
    a.q.fill_(1.0)
    ref, bound = tight(a)
    a.run(samhip, gpu_ctx)
    a.verify(ref, bound)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("exponent", [4, 10, 12, 13, 14, 16, 20, 40, 90, 100])
def test_scores_whose_f32_numbers_lie_far_apart(samhip, gpu_ctx, exponent, rows, hd):
    """Scores up to 2^117 of either sign, a hundredth of themselves or more apart,
    each of several keys: a query has the mean of its largest's values.  Weights
    are then 1, products with scales below 2^16 and above 2^-10, so that fp16's
    half step is 2^-25 on codes up to 127; hi + lo and the sums 2^-19."""
    print("far scores", exponent, rows, hd, flush=True)
    m, heads = 700, 2
    for sign in (1, -1):
        p = Pages([rows], [m], 1, hd, False, 41, seed=53).fill(53)
        level = 1 + 37 * torch.arange(m, device="cuda") % 100
        k = (127.0 * level)[:, None].expand(m, hd).contiguous()   # scales of whole numbers, codes of 127
        p.caches[0][p.at(0, range(m))] = torch.as_tensor(packed(k, False), device="cuda")
        a = Attend(p, heads, True, seed=53)
        a.q.fill_(sign * 2.0 ** exponent)
        a.q[:, hd:] *= -1
        v = values(p.caches[1][p.at(0, range(m))], False)
        ref = torch.zeros_like(a.out, dtype=torch.float64)
        for i in range(rows):
            seen = level[:m - rows + 1 + i]
            for h in range(heads):
                s = seen if (sign > 0) == (h == 0) else -seen
                if exponent < 10:   # weights of others too
                    w = torch.softmax(s.double() * (127 * hd * a.scale * 2.0 ** exponent), -1)
                else:
                    w = (s == s.max()).double() / (s == s.max()).sum()
                ref[i, h * hd:(h + 1) * hd] = w @ v[:len(seen)]
        a.run(samhip, gpu_ctx)
        a.verify(ref, torch.full_like(ref, 127 * 2.0 ** -25 + 4 * 2.0 ** -19))


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("above", [20.0, 45.0, 60.0])
def test_a_key_of_nearly_all_the_weight_without_values(samhip, gpu_ctx, above, rows, hd, q4):
    """Values of zeros at a key `above` nats over the others: what is left is theirs, to its last digits."""
    p = Pages([rows], [300], 1, hd, q4, 64, seed=54).fill(54)
    k = torch.zeros(300, hd, device="cuda")
    k[100] = above / hd
    p.caches[0][p.at(0, range(300))] = torch.as_tensor(packed(k, q4), device="cuda")
    scale_blocks(p, 0, 1, [100], 0.0)
    a = Attend(p, 2, seed=54, scale=1.0)
    a.q.fill_(1.0)
    ref, bound = tight(a)
    a.run(samhip, gpu_ctx)
    a.verify(ref, bound)


def test_lengths_past_the_last_position_there_may_be(samhip, gpu_ctx):
    """Tables of 2^30 positions, lengths beyond: rows stand where the length says,
    so that some have no place, and the others' queries see up to their own."""
    page, n = 1 << 26, 10
    p = Pages([n], [1], 1, 32, True, 16, seed=55)
    p.page, p.max_pages = page, 16
    p.pages = ints([[-1] * 15 + [0]])
    p.caches = [torch.zeros(page, 18, dtype=torch.uint8, device="cuda") for _ in "kv"]
    k, v = (torch.randn(n, 32, device="cuda") for _ in "kv")
    for over in (5, 9, 10, 2 ** 30 - 1):
        lost = min(n, over)   # the last rows', from position 2^30 on
        p.len = ints([2 ** 30 + over])
        for c in p.caches:
            c[-64:] = 0
        out = [torch.full_like(k, 7.0) for _ in "kv"]
        torch.cuda.synchronize()
        gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, v))
        gpu_ctx.cache_read(p.desc(samhip), *(describe(samhip, o) for o in out))
        gpu_ctx.synchronize()
        for x, o, c in zip((k, v), out, p.caches):
            bytes_ = torch.as_tensor(packed(x, True), device="cuda")
            want = torch.zeros_like(c[-64:])
            if lost < n:   # row i at 2^30 + over - n + i, the last page's
                at = 64 + over - n
                want[at:at + n - lost] = bytes_[:n - lost]
            assert torch.equal(c[-64:], want)
            back = values(bytes_, True)
            back[n - lost:] = 0.0
            assert torch.equal(o.double(), back)
        if over != 5:
            continue
        # keys of zeros: a query has the mean of the values up to its position
        p.caches[0].zero_()
        a = Attend(p, 1, True, seed=55)
        a.max_len = 2 ** 31 - 1
        a.run(samhip, gpu_ctx)
        stored = values(p.caches[1][-64:], True)
        for i in range(n):
            last = min(2 ** 30, 2 ** 30 + over - n + i + 1)   # positions below it are seen
            count = last - (2 ** 30 - page)
            want = stored[:64 - (2 ** 30 - last)].sum(0) / count
            assert ((a.out[i].double() - want).abs() <= 1e-5 * stored.abs().sum(0) / count + 2.0 ** -40).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_no_scratch_where_no_keys_are_split(samhip, rows):
    """So many kv heads that every workgroup has all keys of its queries: nothing is kept for a join."""
    with samhip.Context(0) as ctx:
        p = Pages([rows], [600], 4096, 32, True, 64, seed=56)
        x = torch.randn(600, p.width, device="cuda")
        for c in p.caches:
            for at in range(0, 600, 100):
                c[p.at(0, range(at, at + 100))] = torch.as_tensor(packed(x[at:at + 100], True), device="cuda")
        a = Attend(p, 4096, seed=56)
        a.run(samhip, ctx)
        assert ctx.query().activation_allocation_peak_bytes == 0
        k = values(p.caches[0][p.at(0, range(600))], True).view(600, 4096, 32).float()
        q = a.q.view(rows, 4096, 32)
        w = torch.softmax(torch.bmm(q.transpose(0, 1).contiguous(), k.permute(1, 2, 0).contiguous()) * a.scale, -1)
        want = torch.bmm(w, k.transpose(0, 1).contiguous()).transpose(0, 1).reshape(rows, -1)
        assert ((a.out - want).abs() <= 1e-4).all()


@pytest.mark.parametrize("q4", [False, True])
def test_rows_with_one_place_mix_there_alone(samhip, gpu_ctx, q4):
    """Requests whose pages are the same in one call: of what stands there each byte
    is one of theirs, every other place holds its own row."""
    n = 600   # several workgroups' rows
    p = Pages([n, n, n], [n, n, n], 4, 64, q4, 16, seed=58)
    table = p.table.copy()
    table[2] = table[0]
    p.pages.copy_(ints(table.tolist()))
    k, v = (torch.randn(p.rows, p.width, device="cuda") for _ in "kv")
    torch.cuda.synchronize()
    gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, v))
    gpu_ctx.synchronize()
    for x, c in zip((k, v), p.caches):
        bytes_ = torch.as_tensor(packed(x, q4), device="cuda")
        shared, own = c[p.at(0, range(n))], c[p.at(1, range(n))]
        assert torch.equal(own, bytes_[n:2 * n])
        assert ((shared == bytes_[:n]) | (shared == bytes_[2 * n:])).all()
        nobody = torch.ones(len(c), dtype=torch.bool, device="cuda")
        nobody[torch.cat([p.at(0, range(n)), p.at(1, range(n))])] = False
        assert (c[nobody] == 255).all()


def test_q8_0_codes_at_ties_are_of_one_division(samhip, gpu_ctx):
    """Values next to ties whose code follows from 127 / amax as one division, and
    is another by a product with a rounded 1 / amax."""
    rng = np.random.default_rng(57)
    most = rng.uniform(0.5, 4, 1 << 16).astype(np.float32)
    once, twice = np.float32(127) / most, np.float32(127) * (np.float32(1) / most)
    x = ((rng.integers(0, 120, (1 << 16, 31)) + 0.5) / once[:, None]).astype(np.float32)
    x = np.concatenate([most[:, None], x], 1)   # the largest first
    other = np.rint(x * twice[:, None]) != np.rint(x * once[:, None])
    x = x[other.any(1)]
    x = x[:len(x) // 2 * 2].reshape(-1, 64)
    assert len(x) > 1000
    p = Pages([len(x)], [len(x)], 2, 32, False, 16, seed=57)
    k = torch.as_tensor(x, device="cuda")
    torch.cuda.synchronize()
    gpu_ctx.cache_write(p.desc(samhip), None, describe(samhip, k), describe(samhip, k))
    gpu_ctx.synchronize()
    want = packed(k, False)
    for c in p.caches:
        assert np.array_equal(c[p.at(0, range(len(x)))].cpu().numpy(), want)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("rows,hd", [(1, 32), (3, 128), (40, 64), (40, 128), (70, 32)])
def test_large_scores_give_means_of_values(samhip, gpu_ctx, rows, hd, q4):
    """Random scores from 2^18 to 2^40 and past, in one part of keys and in several:
    values between 1 and 2, so that every output lies between the smallest and the
    largest of its dimension, but for what the bound leaves (a unit of code is at
    most a seventh, 2^-25 of the largest weight for each key)."""
    lens = [3000, 97]
    for e in range(12, 36):
        print("large scores", e, rows, hd, q4, flush=True)
        p = Pages([rows, rows], lens, 2, hd, q4, 41, seed=59).fill(59)
        g = torch.Generator(device="cuda").manual_seed(e)
        for r, m in enumerate(lens):
            x = 1 + torch.rand(m, p.width, device="cuda", generator=g)
            p.caches[1][p.at(r, range(m))] = torch.as_tensor(packed(x, q4), device="cuda")
        a = Attend(p, 4, True, seed=e)
        a.q.mul_(2.0 ** e)
        a.run(samhip, gpu_ctx)
        for r, m in enumerate(lens):
            v = values(p.caches[1][p.at(r, range(m))][:, :p.row_bytes], q4).view(m, 2, hd)
            for i in range(rows):
                seen = v[:m - rows + 1 + i]
                lo, hi = (t.repeat_interleave(2, 0) for t in (seen.amin(0), seen.amax(0)))
                out = a.out[p.starts[r] + i].double().view(4, hd)
                slack = len(seen) * 16 * 2.0 ** -25 + 2.0 ** -16
                assert ((out >= lo - slack) & (out <= hi + slack)).all(), (r, i)
