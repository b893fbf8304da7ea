"""The operators of a batch of requests on one image, run together as a
service would: the image's map through group norm, its keys and values and
the requests' queries and own keys through packed projections with adapters
beside them, attention to the shared prefix and the own keys, and the output
projection.

Each new operator is checked on the inputs it has in the run, against its
definition in F64 on the card (the packed products between them are
samhip_mul_mat's, checked elsewhere).  Tolerances, relative L2: group norm
with erf-GELU 1e-6 (F32 steps on F64 statistics), adapters 1e-6 (F32 sums of
at most 256 products and 16 ranks: random signs leave them below
sqrt(256) 2^-24 = 1e-6), attention 1e-5 (operands of ~22 bits, scores below
30: 30 * 2^-21).  Then the whole run is captured and replayed on new inputs;
a replay gives the eager run's bits."""

import numpy as np
import pytest

try:
    import torch
except ImportError:   # pragma: no cover
    torch = None

pytestmark = pytest.mark.gpu

C, HEADS, HD, GROUPS, RANK, SLOTS = 256, 8, 32, 8, 16, 5
SIDE, PROMPTS, QUERIES, OWN = 24, [3, 0, 4, 1], 201, 33


def describe(samhip, t):
    return samhip.tensor_nd(samhip.F16 if t.dtype == torch.float16 else samhip.F32, t.shape[::-1],
                            [v * t.element_size() for v in t.stride()[::-1]], t.data_ptr())


def rel(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


class Service:
    def __init__(self, samhip, ctx):
        self.sh, self.ctx = samhip, ctx
        g = torch.Generator(device="cuda").manual_seed(1)
        rand = lambda *s, std=1.0: torch.randn(*s, device="cuda", generator=g) * std  # noqa: E731
        self.g = g
        rng = np.random.default_rng(2)
        self.weights = {n: ctx.upload(ctx.quantize(samhip.Q8_0, (rng.standard_normal((C, C)) * 0.06).astype(np.float32))) for n in "qkvo"}
        self.banks = {n: (rand(SLOTS, RANK, C, std=C ** -0.5).half(), rand(SLOTS, C, RANK, std=0.3).half()) for n in "qkvo"}
        self.scales = torch.rand(SLOTS, device="cuda", generator=g) + 0.5
        n_req, rows, own = len(PROMPTS), len(PROMPTS) * QUERIES, len(PROMPTS) * OWN
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        per_row = lambda n: ints([s for s in PROMPTS for _ in range(n)])  # noqa: E731
        self.ids = {"image": ints([2] * (SIDE * SIDE)), "queries": per_row(QUERIES), "own": per_row(OWN)}
        self.q_start, self.own_start = ints([QUERIES * i for i in range(n_req + 1)]), ints([OWN * i for i in range(n_req)])
        self.own_len = ints([33, 2, 17, 0])
        self.w, self.b = rand(C, std=0.2) + 1, rand(C, std=0.2)
        empty = lambda n: torch.empty(n, C, device="cuda")  # noqa: E731
        self.map, self.prompt, self.query = torch.empty(1, SIDE * SIDE, C, device="cuda"), empty(own), empty(rows)
        self.t = {n: empty(SIDE * SIDE) for n in ("tokens", "pk", "pv")} | {n: empty(own) for n in ("ok", "ov")} | {n: empty(rows) for n in ("q", "a", "o")}
        self.new_inputs()

    def new_inputs(self):
        self.map.normal_(0.5, 2.0, generator=self.g)
        self.prompt.normal_(generator=self.g)
        self.query.normal_(generator=self.g)

    def project(self, weight, x, ids, y, after=None):
        sh = self.sh
        self.ctx.mul_mat(sh.tensor(sh.Q8_0, C, C, self.weights[weight].ptr), describe(sh, x), describe(sh, y))
        if after:
            after("base", y)
        a, b = self.banks[weight]
        bank = sh.lora_bank(describe(sh, a), describe(sh, b), None, self.scales.data_ptr())
        self.ctx.lora_add(bank, describe(sh, x), sh.tensor(sh.I32, x.shape[0], 1, ids.data_ptr()), describe(sh, y), describe(sh, y))
        if after:
            after(weight, x, ids, y)

    def run(self, after=None):
        sh, t = self.sh, self.t
        self.ctx.group_norm(describe(sh, self.map), describe(sh, t["tokens"].view(1, -1, C)), GROUPS, self.w.data_ptr(), self.b.data_ptr(), 1e-5,
                            sh.ACT_GELU_ERF)
        self.project("k", t["tokens"], self.ids["image"], t["pk"], after)
        self.project("v", t["tokens"], self.ids["image"], t["pv"], after)
        self.project("k", self.prompt, self.ids["own"], t["ok"], after)
        self.project("v", self.prompt, self.ids["own"], t["ov"], after)
        self.project("q", self.query, self.ids["queries"], t["q"], after)
        self.ctx.prefix_attn(sh.prefix_attn_desc(
            HEADS, HEADS, HD, HD ** -0.5, describe(sh, t["q"]), describe(sh, t["a"]), describe(sh, t["pk"]), describe(sh, t["pv"]), describe(sh, t["ok"]),
            describe(sh, t["ov"]), len(PROMPTS), self.q_start.data_ptr(), self.own_start.data_ptr(), self.own_len.data_ptr(), OWN))
        self.project("o", t["a"], self.ids["queries"], t["o"], after)

    def check_adapters(self, *said):
        self.ctx.synchronize()
        if said[0] == "base":
            self.base = said[1].double()
            return
        weight, x, ids, y = said
        a, b = self.banks[weight]
        want = self.base.clone()
        for s in range(SLOTS):
            m = ids == s
            want[m] += self.scales[s].double() * (x[m].double() @ a[s].double().t() @ b[s].double().t())
        assert rel(y, want) < 1e-6, weight

    def check_rest(self):
        t = self.t
        x = self.map.double().view(-1, GROUPS, C // GROUPS)
        y = ((x - x.mean((0, 2), keepdim=True)) / torch.sqrt(x.var((0, 2), correction=0, keepdim=True) + 1e-5)).reshape(-1, C)
        y = y * self.w.double() + self.b.double()
        assert rel(t["tokens"], 0.5 * y * (1 + torch.erf(y / 2 ** 0.5))) < 1e-6
        want = torch.empty_like(t["a"], dtype=torch.float64)
        for r, n in enumerate(self.own_len.tolist()):
            q = t["q"][r * QUERIES:(r + 1) * QUERIES].double().view(-1, HEADS, HD).transpose(0, 1)
            k, v = (torch.cat([t["p" + x], t["o" + x][r * OWN:r * OWN + n]]).double().view(-1, HEADS, HD).transpose(0, 1).contiguous() for x in "kv")
            s = q @ k.transpose(1, 2).contiguous() * HD ** -0.5
            assert s.abs().max().item() < 30
            want[r * QUERIES:(r + 1) * QUERIES] = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(-1, C)
        assert rel(t["a"], want) < 1e-5


def test_run_of_a_request_batch(samhip):
    with samhip.Context(0) as ctx:
        s = Service(samhip, ctx)
        torch.cuda.synchronize()
        s.run(after=s.check_adapters)
        ctx.synchronize()
        s.check_rest()
        s.run()   # every product and operator has its staging
        ctx.capture_begin()
        s.run()
        graph = ctx.capture_end()
        for _ in range(3):
            s.new_inputs()
            torch.cuda.synchronize()
            s.run()
            ctx.synchronize()
            eager = {n: v.clone() for n, v in s.t.items()}
            for v in s.t.values():
                v.zero_()
            torch.cuda.synchronize()
            graph.launch()
            ctx.synchronize()
            for n, v in s.t.items():
                assert torch.equal(v, eager[n]), n
        graph.destroy()


def test_runs_on_the_callers_stream(samhip):
    """The operators run on the context's current stream, in its order: work
    that a side stream has not finished yet is waited for by the stream alone."""
    with samhip.Context(0) as ctx:
        s = Service(samhip, ctx)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        s.run()
        ctx.synchronize()
        want = {n: v.clone() for n, v in s.t.items()}
        keep = [v.clone() for v in (s.map, s.prompt, s.query)]
        for v in (s.map, s.prompt, s.query):
            v.zero_()
        torch.cuda.synchronize()
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(4):
                big = big @ big * 1e-3
            for v, k in zip((s.map, s.prompt, s.query), keep):
                v.copy_(k)
        s.run()
        with torch.cuda.stream(stream):
            got = {n: v.clone() for n, v in s.t.items()}
        stream.synchronize()
        for n in want:
            assert torch.equal(got[n], want[n]), n
        ctx.set_stream(None)


def test_a_switch_of_streams_orders_the_calls(samhip):
    """Calls on one stream, still waiting behind other work, share the context's
    scratch with those made on the next: the next stream waits."""
    with samhip.Context(0) as ctx:
        s = Service(samhip, ctx)
        inputs = []
        for _ in range(3):
            s.new_inputs()
            inputs.append([v.clone() for v in (s.map, s.prompt, s.query)])
        want = []
        for given in inputs:
            for v, k in zip((s.map, s.prompt, s.query), given):
                v.copy_(k)
            torch.cuda.synchronize()
            s.run()
            ctx.synchronize()
            want.append({n: v.clone() for n, v in s.t.items()})
        services = [Service(samhip, ctx) for _ in inputs]
        streams = [torch.cuda.Stream() for _ in inputs[:2]] + [None]
        for each, given in zip(services, inputs):
            for v, k in zip((each.map, each.prompt, each.query), given):
                v.copy_(k)
        big = torch.randn(4096, 4096, device="cuda")
        torch.cuda.synchronize()
        for each, stream in zip(services, streams):
            if stream:
                with torch.cuda.stream(stream):
                    held = big
                    for _ in range(4):
                        held = held @ big * 1e-3
            ctx.set_stream(stream.cuda_stream if stream else None)
            each.run()
        ctx.synchronize()   # the last stream, behind both others
        for each, expected in zip(services, want):
            for n in expected:
                assert torch.equal(each.t[n], expected[n]), n
