"""samhip_prefix_attn against its definition in F64.

Tolerance, for every output element, from the arithmetic: operands enter the
products as hi + lo fp16 halves (off by 2^-22 of the value, the dropped
lo * lo another 2^-22), sums are F32.  A score is off by at most
  ds = scale sum|q||k| (head_dim 2^-24 + 5 * 2^-22),
a weight relative to the others by 2 ds + 2^-21 (exp2 and its argument's
rounding are within it), P and V add 4 * 2^-22, and the sums over n keys run
in chains of at most n / 16 + 48 steps.  So
  |error| <= sum w|v| (2 ds + 2^-19 + (n / 16 + 48) 2^-24)."""

import ctypes

import pytest

try:
    import torch
except ImportError:   # pragma: no cover
    torch = None


def describe(samhip, t):
    return samhip.tensor_nd(samhip.F16 if t.dtype == torch.float16 else samhip.F32, t.shape[::-1],
                            [v * t.element_size() for v in t.stride()[::-1]], t.data_ptr())


def strided(t, pad, dtype):
    held = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), device=t.device, dtype=dtype)
    held[:, :t.shape[1]] = t
    return held[:, :t.shape[1]]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Batch:
    """Inputs of one call: q_len and own_len per request, own rows in slots of
    `own_max + gap` rows, NaN wherever nothing may be read."""

    def __init__(self, q_len, prefix, own_len, heads, kv_heads, hd, dtype, causal=False, pad=0, seed=0, first=0, behind=0, gap=1, amp=1.0, own_max=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        dt = torch.float16 if dtype == "f16" else torch.float32
        self.q_len, self.own_len, self.prefix, self.heads, self.kv_heads, self.hd, self.causal = q_len, own_len, prefix, heads, kv_heads, hd, causal
        self.scale = hd ** -0.5
        self.own_max = max(own_len) if own_max is None else own_max
        self.first, rows = first, first + sum(q_len) + behind
        self.q = strided(rand(rows, heads * hd) * amp, pad, torch.float32)
        w = kv_heads * hd
        self.pk, self.pv = strided(rand(prefix, w) * amp + 0.2, pad, dt), strided(rand(prefix, w), pad, dt)
        slot = max(own_len + [0]) + gap
        self.slot = slot
        self.ok, self.ov = strided(rand(len(q_len) * slot, w) * amp, pad, dt), strided(rand(len(q_len) * slot, w), pad, dt)
        for r, n in enumerate(own_len):
            self.ok[r * slot + n:(r + 1) * slot] = float("nan")
            self.ov[r * slot + n:(r + 1) * slot] = float("nan")
        self.starts = [first + sum(q_len[:i]) for i in range(len(q_len) + 1)]
        self.q_start, self.own_start, self.lens = ints(self.starts), ints([r * slot for r in range(len(q_len))]), ints(own_len)
        self.held = torch.full((rows, heads * hd + pad), 7.0, device="cuda")
        self.out = self.held[:, :heads * hd]

    def desc(self, samhip):
        d = lambda t: describe(samhip, t)  # noqa: E731
        return samhip.prefix_attn_desc(self.heads, self.kv_heads, self.hd, self.scale, d(self.q), d(self.out), d(self.pk), d(self.pv), d(self.ok),
                                       d(self.ov), len(self.q_len), self.q_start.data_ptr(), self.own_start.data_ptr(), self.lens.data_ptr(),
                                       self.own_max, self.causal)

    def reference(self):
        h, hd, group = self.heads, self.hd, self.heads // self.kv_heads
        ref = torch.full((self.q.shape[0], h * hd), 7.0, device="cuda", dtype=torch.float64)
        bound = torch.zeros_like(ref)
        for r, n in enumerate(self.q_len):
            if not n:
                continue
            m, s0 = self.own_len[r], self.starts[r]
            q = self.q[s0:s0 + n].double().view(n, h, hd)
            at = r * self.slot
            k = torch.cat([self.pk, self.ok[at:at + m]]).double().view(-1, self.kv_heads, hd)
            v = torch.cat([self.pv, self.ov[at:at + m]]).double().view(-1, self.kv_heads, hd)
            keys = k.shape[0]
            seen = torch.ones(n, keys, dtype=torch.bool, device="cuda")
            if self.causal:
                i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")[None, :]
                seen[:, self.prefix:] = j <= i + (m - n)
            for head in range(h):
                kk, vv = k[:, head // group], v[:, head // group]
                s = (q[:, head] @ kk.t()) * self.scale
                mag = (q[:, head].abs() @ kk.abs().t()) * self.scale
                s = s.masked_fill(~seen, -torch.inf)
                some = seen.any(1, keepdim=True)
                top = s.amax(1, keepdim=True) if keys else s.new_zeros(n, 1)
                w = torch.where(seen, torch.exp(s - torch.where(some, top, 0.0)), 0.0)
                w = w / torch.where(some, w.sum(1, keepdim=True), 1.0)
                cols = slice(head * hd, (head + 1) * hd)
                ref[s0:s0 + n, cols] = w @ vv
                ds = (mag.masked_fill(~seen, 0.0).amax(1, keepdim=True) if keys else 0.0) * (hd * 2.0 ** -24 + 5 * 2.0 ** -22)
                bound[s0:s0 + n, cols] = (w @ vv.abs()) * (2 * ds + 2.0 ** -19 + (keys / 16 + 48) * 2.0 ** -24)
        return ref, bound

    def check(self, samhip, ctx):
        ref, bound = self.reference()
        torch.cuda.synchronize()
        ctx.prefix_attn(self.desc(samhip))
        ctx.synchronize()
        self.verify(ref, bound)

    def verify(self, ref, bound):
        err = (self.out.double() - ref).abs()
        assert (err <= bound).all(), (err / bound.clamp(min=1e-30)).max().item()
        assert (self.held[:, self.heads * self.hd:] == 7.0).all()


# query lengths, prefix, own lengths, heads, kv heads
CASES = [
    ([1], 1, [0], 1, 1),
    ([1], 0, [1], 2, 1),
    ([1] * 8, 5184, [0, 64, 1, 33, 2, 40, 31, 32], 8, 8),
    ([201] * 3, 577, [33, 2, 0], 8, 8),
    ([1] * 70, 300, [(7 * i) % 150 for i in range(70)], 8, 2),
    ([5, 0, 150, 31, 0, 1, 64], 1000, [9, 3, 300, 31, 0, 77, 64], 12, 4),
    ([3, 40], 0, [0, 50], 4, 4),
    ([2, 3], 31, [0, 0], 16, 1),
    ([9] * 5, 129, [700, 1, 256, 257, 0], 3, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_prefix_attn(samhip, gpu_ctx, case, hd, dtype):
    q_len, prefix, own_len, heads, kv_heads = CASES[case]
    print(f"prefix_attn {CASES[case]} hd={hd} {dtype}", flush=True)
    for causal in (False, True):
        Batch(q_len, prefix, own_len, heads, kv_heads, hd, dtype, causal=causal, pad=(0, 3)[causal], seed=case, first=(0, 2)[causal],
              behind=(0, 3)[causal]).check(samhip, gpu_ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_peaked_scores(samhip, gpu_ctx, dtype):
    """Scores of hundreds: one key takes all the weight, the running maximum moves."""
    Batch([40, 7], 2000, [65, 200], 4, 2, 64, dtype, causal=True, amp=6.0, seed=3).check(samhip, gpu_ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [-60, -30, 30, 45])
def test_f32_keys_and_values_of_any_magnitude(samhip, gpu_ctx, exponent):
    """Keys of 2^e against queries of 2^-e, values of 2^e, one tile of values
    2^20 times larger than the rest."""
    b = Batch([33, 1], 260, [40, 3], 4, 4, 64, "f32", seed=4)
    b.q.mul_(2.0 ** -exponent)
    for t in (b.pk, b.ok, b.pv, b.ov):
        t.mul_(2.0 ** exponent)
    b.pv[128:160].mul_(2.0 ** 20)
    b.check(samhip, gpu_ctx)


@pytest.mark.gpu
def test_zero_keys_values_and_queries(samhip, gpu_ctx):
    b = Batch([33, 1], 260, [40, 3], 4, 4, 32, "f32", seed=4)
    b.pk.zero_()
    b.q[3].zero_()
    b.ov.nan_to_num_(0.0)
    b.ov.zero_()
    b.check(samhip, gpu_ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 200])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_non_finite_keys_reach_only_queries_that_see_them(samhip, gpu_ctx, dtype, hd, prefix):
    """Query i of 40 sees own keys up to i + 30 of 70: key 50 holds a NaN in kv
    head 0, value 61 an infinity in kv head 1, value 69 both."""
    b = Batch([40, 3], prefix, [70, 3], 4, 2, hd, dtype, causal=True, seed=13)
    ref, bound = b.reference()
    b.ok[50, 5] = float("nan")
    b.ov[61, hd + 7] = float("inf")
    b.ov[69, hd - 1] = float("-inf")
    b.ov[69, hd] = float("nan")
    torch.cuda.synchronize()
    gpu_ctx.prefix_attn(b.desc(samhip))
    gpu_ctx.synchronize()
    sees = torch.zeros(43, 4, dtype=torch.bool, device="cuda")   # by query and head
    sees[20:40, :2] = True
    sees[31:40, 2:] = True
    out = b.out.view(43, 4, hd)
    err, most = (out.double() - ref.view(43, 4, hd)).abs(), bound.view(43, 4, hd)
    assert (err[~sees] <= most[~sees]).all(), (err[~sees] / most[~sees]).max().item()
    assert not out[sees].isfinite().all(-1).any()


@pytest.mark.gpu
def test_tables_out_of_range_are_cut(samhip, gpu_ctx):
    """Lengths and starts beyond the buffers: nothing outside them is read."""
    b = Batch([4, 4, 4, 4], 50, [10, 10, 10, 10], 2, 2, 32, "f16", seed=9, gap=0)
    b.own_start.copy_(ints([0, -5, 35, 2 ** 31 - 1]))
    b.lens.copy_(ints([-3, 10, 1000, 10]))
    b.own_max = 2 ** 30
    b.q_start.copy_(ints([-7, 4, 8, 12, 2 ** 31 - 1]))
    ref = Batch([4, 4, 4, 4], 50, [0, 0, 5, 0], 2, 2, 32, "f16", seed=9, gap=5)
    ref.q, ref.pk, ref.pv = b.q, b.pk, b.pv
    ref.ok[20:25], ref.ov[20:25] = b.ok[35:40], b.ov[35:40]
    want, bound = ref.reference()
    torch.cuda.synchronize()
    gpu_ctx.prefix_attn(b.desc(samhip))
    gpu_ctx.synchronize()
    b.verify(want, bound)


@pytest.mark.gpu
def test_captured_replays_follow_the_tables(samhip, gpu_ctx):
    """One graph, replayed as the requests' caches grow and their queries move."""
    b = Batch([1] * 6, 700, [20] * 6, 8, 4, 64, "f16", causal=True, seed=11, own_max=20)
    b.check(samhip, gpu_ctx)
    keep_k, keep_v = b.ok.nan_to_num(0.0), b.ov.nan_to_num(0.0)
    gpu_ctx.capture_begin()
    gpu_ctx.prefix_attn(b.desc(samhip))
    graph = gpu_ctx.capture_end()
    for step, lens in enumerate(([0, 1, 2, 3, 4, 5], [20, 19, 0, 7, 7, 7], [1] * 6, [20] * 6)):
        b.q.normal_()
        b.own_len = lens
        b.lens.copy_(ints(lens))
        b.ok.copy_(keep_k)
        b.ov.copy_(keep_v)
        b.q_len = [1] * 6 if step % 2 == 0 else [0, 3, 0, 1, 2, 0]
        b.starts = [sum(b.q_len[:i]) for i in range(7)]
        b.q_start.copy_(ints(b.starts))
        b.held.fill_(7.0)
        ref, bound = b.reference()
        torch.cuda.synchronize()
        graph.launch()
        gpu_ctx.synchronize()
        b.verify(ref, bound)
        torch.randn(4096, 256, device="cuda") @ torch.randn(256, 64, device="cuda")
    graph.destroy()


# The two forms of the prefix part, few query places and many, with own keys;
# then calls of one part, which writes the output itself, in either form.
FORMS = [([3], 3000, [40]), ([100, 30], 3000, [200, 3]), ([3], 200, [0]), ([100], 200, [0])]


def change_values(b, change):
    """`change` on the values of the prefix and of each request's own rows."""
    change(b.pv)
    for r, n in enumerate(b.own_len):
        change(b.ov[r * b.slot:r * b.slot + n])


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("exponent", [-30, -60])
@pytest.mark.parametrize("place", [0, 2])
def test_zero_value_rows_beside_small_values(samhip, gpu_ctx, form, exponent, place):
    """64 of every 256 value rows are zero, as padded tokens' are: the others keep their digits."""
    b = Batch(*FORMS[form], 4, 4, 64, "f32", seed=20)

    def change(v):
        v.mul_(2.0 ** exponent)
        v[torch.arange(v.shape[0], device="cuda") // 64 % 4 == place] = 0.0
    change_values(b, change)
    b.check(samhip, gpu_ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("exponent", [112, 124])
def test_f32_values_near_the_largest(samhip, gpu_ctx, form, exponent):
    """Values to 5 * 2^exponent: their weighted mean fits, whatever their sum does."""
    b = Batch(*FORMS[form], 4, 2, 32, "f32", seed=24)
    change_values(b, lambda v: v.mul_(2.0 ** exponent))
    b.check(samhip, gpu_ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,prefix", [(1, 65536), (40, 1024), (4096, 5184)])
@pytest.mark.parametrize("below", [16.75, 17.5, 18.5])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_many_small_weights_behind_a_large_one(samhip, gpu_ctx, dtype, rows, prefix, below):
    """The first key's score is `below` nats above all others', and all values
    are one: the output is one.  Scores are exact (queries 1, keys a multiple of
    2^-14), numerator and denominator have the same weights, so what counts is
    the split of the weights (2^-22 of each, 2^-36 of the largest at least) and
    the F32 sums: 2^-19 + prefix 2^-36 + (prefix / 16 + 48) 2^-24."""
    heads, hd = 8, 32
    b = Batch([rows], prefix, [0], heads, heads, hd, dtype, seed=25)
    b.scale = 0.125
    b.q.fill_(1.0)
    b.pk.zero_()
    b.pk[0] = below / (hd * b.scale)
    b.pv.fill_(1.0)
    torch.cuda.synchronize()
    gpu_ctx.prefix_attn(b.desc(samhip))
    gpu_ctx.synchronize()
    err = (b.out.double() - 1).abs().max().item()
    assert err <= 2.0 ** -19 + prefix * 2.0 ** -36 + (prefix / 16 + 48) * 2.0 ** -24, err


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("large,key", [(2.0 ** 33, -5.0), (2.0 ** 40, -5.0), (3e38, -24.0)])
@pytest.mark.parametrize("place", [0, 70, 199])
def test_large_values_without_weight(samhip, gpu_ctx, form, large, key, place):
    """One value row of the prefix and one of the first request's own are far
    larger than all others, at a weight (a score 44 or 210 below the others, at
    least) that leaves little or nothing of them.  The rest of their 64 rows are
    zero; the rows of other tiles keep their digits."""
    b = Batch(*FORMS[form], 4, 4, 64, "f32", seed=21)
    b.q.abs_().add_(0.5)
    for k, v, n in ((b.pk, b.pv, b.prefix), (b.ok, b.ov, b.own_len[0])):
        if place < n:
            v[place // 64 * 64:min(place // 64 * 64 + 64, n)] = 0.0
            v[place] = large
            k[place] = key
    b.check(samhip, gpu_ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("large", [2.0 ** 40, 1e30])
def test_a_large_dimension_leaves_the_others(samhip, gpu_ctx, form, large):
    """Dimension 5 of one value row is far larger, at an ordinary weight: so are
    that dimension's results, and the others keep their digits in the rows of
    other tiles (its own 64 are zero), smaller ones among them."""
    b = Batch(*FORMS[form], 4, 2, 64, "f32", seed=22)
    b.pv[64:128] = 0.0
    b.pv[70, 5] = large
    b.pv[130:190].mul_(2.0 ** -30)
    b.check(samhip, gpu_ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_non_finite_values_reach_only_their_dimension(samhip, gpu_ctx, dtype, causal, form):
    """Value 70 of the prefix holds an infinity in dimension 5 of kv head 0, the
    first request's own value 30 a NaN in dimension 9 and own value 33 a -inf in
    dimension 40 of kv head 1 (of 64)."""
    b = Batch(*FORMS[form], 4, 2, 64, dtype, causal=causal, seed=23)
    ref, bound = b.reference()
    b.pv[70, 5] = float("inf")
    reached = torch.zeros(b.q.shape[0], 4, 64, dtype=torch.bool, device="cuda")
    reached[:, :2, 5] = True
    if b.own_len[0]:
        b.ov[30, 64 + 9] = float("nan")
        b.ov[33, 64 + 40] = float("-inf")
        for key, d in ((30, 9), (33, 40)):
            n = b.q_len[0]
            reached[max(0, key - (b.own_len[0] - n)) if causal else 0:n, 2:, d] = True
    torch.cuda.synchronize()
    gpu_ctx.prefix_attn(b.desc(samhip))
    gpu_ctx.synchronize()
    out = b.out.view(-1, 4, 64)
    assert torch.equal(~out.isfinite(), reached)
    err, most = (out.double() - ref.view(-1, 4, 64)).abs(), bound.view(-1, 4, 64)
    assert (err[~reached] <= most[~reached]).all(), (err[~reached] / most[~reached]).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.125, -2.0, 1e-30])
def test_scales_of_either_sign_and_zero(samhip, gpu_ctx, scale, dtype, form):
    b = Batch(*FORMS[form], 4, 2, 64, dtype, causal=True, seed=26)
    b.scale = abs(scale)
    if scale < 0:   # as with the queries' signs turned
        b.q.neg_()
    ref, bound = b.reference()
    if scale < 0:
        b.q.neg_()
    b.scale = scale
    torch.cuda.synchronize()
    gpu_ctx.prefix_attn(b.desc(samhip))
    gpu_ctx.synchronize()
    b.verify(ref, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(2))
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_non_finite_values_count_at_any_weight(samhip, gpu_ctx, dtype, form):
    """The prefix' scores lie 100 and more below the own keys': what its values
    weigh is nothing, but an infinity among them is not."""
    b = Batch(*FORMS[form], 4, 4, 64, dtype, seed=27)
    b.q.abs_().add_(0.5)
    b.pk.fill_(-24.0)
    ref, bound = b.reference()
    b.pv[70, 5] = float("inf")
    torch.cuda.synchronize()
    gpu_ctx.prefix_attn(b.desc(samhip))
    gpu_ctx.synchronize()
    out, ref, bound = (t.view(-1, 4, 64) for t in (b.out, ref, bound))
    assert not out[:, 0, 5].isfinite().any()
    rest = torch.ones_like(out, dtype=torch.bool)
    rest[:, 0, 5] = False
    assert ((out.double() - ref).abs() <= bound)[rest].all()


def test_refusals(samhip):
    L = samhip.lib()

    def ok(heads=8, kv_heads=4, hd=64, rows=10, prefix=100, own=50, type=1, requests=2, own_max=16, scale=0.125, version=1, q_type=0, q_w=None,
           pv_rows=None, ov_type=None, kv_w=None, q_start=0x100, own_start=0x200, q_nb=None, k_data=0x20000, out_rows=None):
        e = 2 if type == 1 else 4
        w, kw = heads * hd if q_w is None else q_w, kv_heads * hd if kv_w is None else kv_w
        q = samhip.tensor_nd(q_type, (w, rows), (4, q_nb or 4 * w), 0x1000)
        out = samhip.tensor_nd(0, (heads * hd, rows if out_rows is None else out_rows), (4, 4 * heads * hd), 0x10000)
        kv = lambda n, t, p: samhip.tensor_nd(t, (kw, n), (2 if t == 1 else 4, (2 if t == 1 else 4) * kw), p)  # noqa: E731
        d = samhip.prefix_attn_desc(heads, kv_heads, hd, scale, q, out, kv(prefix, type, k_data), kv(prefix if pv_rows is None else pv_rows, type, 0x30000),
                                    kv(own, type, 0x40000), kv(own, type if ov_type is None else ov_type, 0x50000), requests, q_start, own_start, 0x300,
                                    own_max)
        d.version = version
        return L.samhip_supports_prefix_attn(ctypes.byref(d))

    assert ok() == 1 and ok(type=0) == 1 and ok(prefix=0, k_data=0) == 1 and ok(own=0) == 1 and ok(own_max=0, own_start=0) == 1 and ok(q_nb=4096) == 1
    for bad in ({"heads": 6}, {"kv_heads": 0}, {"heads": 0}, {"hd": 16}, {"hd": 96}, {"hd": 256}, {"rows": 0}, {"requests": 0}, {"own_max": -1},
                {"scale": float("nan")}, {"scale": float("inf")}, {"version": 2}, {"q_type": 1}, {"q_w": 500}, {"pv_rows": 99}, {"ov_type": 0},
                {"kv_w": 128}, {"q_start": 0}, {"own_start": 0}, {"q_start": 0x102}, {"q_nb": 1000}, {"k_data": 0}, {"type": 8}, {"out_rows": 9}):
        assert ok(**bad) == 0, bad
    assert L.samhip_supports_prefix_attn(None) == 0
    assert L.samhip_prefix_attn(None, None) == samhip.ERR_INVALID_ARGUMENT
