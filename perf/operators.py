"""The operators of a batch of requests on one image, as cases that can be timed and compared: low-rank adapters beside a shared
projection, attention to a shared prefix and to each request's own keys, and group norm with an activation on channels-last maps.

`run` computes each in its plain form, or, where `own` is set, by the calls of sam.cpp_amd/samhip.py that a user makes.  Sizes are those
of the repository's benchmark and tests (image tokens 72 x 72, widths 256, 1024 and 4736, 201 queries, 32 or 33 prompt tokens, neck maps of
36, 72, 144 and 288 pixels a side), or generic ones of the same ranges."""
import importlib.util
import math
import os

import torch

own = False

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_binding = []


def binding():
    """samhip and the context that a program keeps."""
    if not _binding:
        spec = importlib.util.spec_from_file_location("samhip", os.path.join(ROOT, "sam.cpp_amd", "samhip.py"))
        sh = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sh)
        _binding.extend((sh, sh.Context(0)))
    return _binding


# --- cases ------------------------------------------------------------------


def listed():
    return [
        # One token of each of 16 requests, each with another adapter, at the text encoder's width: launches and latency count.
        lora("adapters_16_tokens", 16, 1024, 1024, 16, 32, "single"),
        # Eight prompts of 32 tokens through the text encoder's first MLP linear, an adapter for each.
        lora("adapters_8_prompts", 256, 1024, 4096, 16, 8, "runs"),
        # Rows of many requests in no order, ranks of many sizes, widths that are a multiple of nothing, F32 adapters, strided rows.
        lora("adapters_ragged_f32", 777, 1001, 1359, 40, 24, "scattered", type="f32", ragged=True, pad=7),
        # The image tokens of eight images through a ViT MLP's first linear, an adapter for each image.
        lora("adapters_8_images", 41472, 1024, 4736, 32, 8, "runs"),
        # One query of each of 8 requests on the image tokens and up to 64 keys of their own, from an F16 cache: single-token serving.
        attn("attend_single_f16", 8, 1, 5184, 64, 8, 8, 32, "f16"),
        # Eight prompts' 201 queries on the image tokens and on their own 2 to 33 prompt tokens, F32 keys and values.
        attn("attend_8_prompts_f32", 8, 201, 5184, 33, 8, 8, 32, "f32"),
        # 64 requests, one token each, on a long prefix with grouped heads, and as many as 1024 tokens of their own: long-cache serving.
        attn("attend_long_prefix_f16", 64, 1, 65536, 1024, 16, 4, 128, "f16", causal=True),
        # Requests of 0 to 150 queries that read their own keys causally, behind a prefix that ends inside a tile; F32.
        attn("attend_ragged_causal_f32", 13, 150, 1000, 300, 12, 4, 64, "f32", causal=True, ragged=True),
        # The smallest neck map, one image.
        norm("norm_relu_36", 1, 36 * 36, 256, 8, "f32", "f32", "relu"),
        # The largest neck map, one image.
        norm("norm_relu_288", 1, 288 * 288, 256, 8, "f32", "f32", "relu"),
        # Eight images' maps from the F16 feature cache.
        norm("norm_silu_8x144_f16", 8, 144 * 144, 256, 32, "f16", "f16", "silu"),
        # Channels, groups and pixels that are a multiple of nothing, strided pixels, F16 in and F32 out.
        norm("norm_gelu_odd", 3, 53 * 37, 345, 15, "f16", "f32", "gelu", pad=11),
    ]


def lora(name, rows, k, n, rank, slots, order, type="f16", ragged=False, pad=0):
    c = {"kind": "lora", "rows": rows, "k": k, "n": n, "rank": rank, "slots": slots, "order": order, "type": type, "ragged": ragged, "pad": pad}
    return {"name": name, **c} if name else c


def attn(name, requests, queries, prefix, own_max, heads, kv_heads, head_dim, type, causal=False, ragged=False):
    c = {"kind": "attn", "requests": requests, "queries": queries, "prefix": prefix, "own_max": own_max, "heads": heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "type": type, "causal": causal, "ragged": ragged}
    return {"name": name, **c} if name else c


def norm(name, images, pixels, channels, groups, type, out, act, pad=0, affine=True):
    c = {"kind": "norm", "images": images, "pixels": pixels, "channels": channels, "groups": groups, "type": type, "out": out, "act": act, "pad": pad,
         "affine": affine}
    return {"name": name, **c} if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lora", "attn", "norm"])
    if kind == "lora":
        rows, k, n, rank = _log(rng, 1, 41472), _log(rng, 32, 4736), _log(rng, 32, 4736), _log(rng, 1, 128)
        slots = rng.randint(1, 64)
        # as much memory as the largest listed case, and its products
        rows = max(1, min(rows, 41472 * (1024 + 2 * 4736) // (k + 2 * n), 41472 * 32 * 8 * 5760 // (rank * slots * (k + n))))
        return lora(None, rows, k, n, rank, slots, rng.choice(["single", "runs", "runs", "scattered"]), rng.choice(["f16", "f16", "f32"]),
                    rng.random() < 0.5, rng.choice([0, 0, 1, 4, 32]))
    if kind == "attn":
        single = rng.random() < 0.5
        head_dim, kv_heads, group = rng.choice([32, 64, 128]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 8])
        queries, requests = (1, rng.randint(1, 64)) if single else (_log(rng, 2, 256), rng.randint(1, 12))
        prefix, own_max = rng.choice([0, 1]) if rng.random() < 0.1 else _log(rng, 16, 65536), _log(rng, 1, 1024) - 1
        while queries * requests * kv_heads * group * head_dim * prefix > 64 * 16 * 128 * 65536:
            prefix = prefix // 2 + 1
        return attn(None, requests, queries, prefix, own_max, kv_heads * group, kv_heads, head_dim, rng.choice(["f16", "f32"]), rng.random() < 0.5,
                    not single and rng.random() < 0.7)
    groups, size = rng.choice([1, 3, 8, 8, 16, 32]), rng.randint(1, 24)
    images, pixels = rng.randint(1, 8), _log(rng, 1, 82944)
    pixels = max(1, min(pixels, 165888 * 256 // (images * groups * size)))
    return norm(None, images, pixels, groups * size, groups, rng.choice(["f32", "f32", "f16"]), rng.choice(["f32", "f32", "f16"]),
                rng.choice(["none", "relu", "silu", "gelu"]), rng.choice([0, 0, 0, 1, 8]), rng.random() < 0.8)


# --- what the cases' lengths and orders are (the same for every seed) ---------


def spread(i, lo, hi):
    """The i-th of numbers spread over lo .. hi."""
    return lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + 0.37) % 1.0))


def rows_slots(case):
    """Each row's slot before the seed turns them: about one request in eight has no adapter (-1)."""
    rows, slots = case["rows"], case["slots"]
    if case["order"] == "runs":  # about as many requests as slots, of uneven lengths
        at, r, ids = 0, 0, []
        while at < rows:
            length = max(1, spread(r, rows // (2 * slots), rows // slots + 1))
            ids += [-1 if r % 8 == 5 else r % slots] * min(length, rows - at)
            at, r = at + length, r + 1
        return ids
    if case["order"] == "single":
        return [-1 if m % 8 == 5 else m % slots for m in range(rows)]
    return [-1 if (s := spread(m, 0, slots)) == slots else s for m in range(rows)]


def slot_rank(case, s):
    return spread(s, 1, case["rank"]) if case["ragged"] else case["rank"]


def query_lengths(case):
    return [spread(r, 0, case["queries"]) if case["ragged"] else case["queries"] for r in range(case["requests"])]


def own_lengths(case):
    """A causal request's own keys hold its queries' at least."""
    return [min(case["own_max"], max(spread(r, 2 * (case["own_max"] >= 33), case["own_max"]), q if case["causal"] else 0))
            for r, q in enumerate(query_lengths(case))]


def work(case):
    if case["kind"] == "lora":
        ids = [s for s in rows_slots(case) if s >= 0]
        each = 2 if case["type"] == "f16" else 4
        used = sum(slot_rank(case, s) for s in set(ids))
        return {"bytes": 4 * len(ids) * case["k"] + 8 * case["rows"] * case["n"] + each * used * (case["k"] + case["n"]) + 4 * case["rows"],
                "flops": 2 * sum(slot_rank(case, s) for s in ids) * (case["k"] + case["n"])}
    if case["kind"] == "attn":
        each = 2 if case["type"] == "f16" else 4
        q, o = query_lengths(case), own_lengths(case)
        keys = 0
        for n, m in zip(q, o):
            keys += n * case["prefix"]
            keys += sum(max(0, m - n + 1 + i) for i in range(n)) if case["causal"] else n * m
        return {"bytes": 8 * sum(q) * case["heads"] * case["head_dim"] + 2 * each * (case["prefix"] + sum(o)) * case["kv_heads"] * case["head_dim"],
                "flops": 4 * keys * case["heads"] * case["head_dim"]}
    n = case["images"] * case["pixels"] * case["channels"]
    return {"bytes": n * ((2 if case["type"] == "f16" else 4) + (2 if case["out"] == "f16" else 4)), "flops": 10 * n}


# --- inputs ------------------------------------------------------------------

DTYPE = {"f32": torch.float32, "f16": torch.float16}


def inputs(case, seed):
    """Tensors by name, from the seed alone; strided ones hold NaN between their rows."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, device=DEV, generator=g) * std + mean

    def strided(t, pad, dtype=torch.float32):
        if not pad:
            return t.to(dtype)
        held = torch.full((*t.shape[:-1], t.shape[-1] + pad), math.nan, device=DEV, dtype=dtype)
        held[..., :t.shape[-1]] = t
        return held[..., :t.shape[-1]]

    if case["kind"] == "lora":
        m, k, n, r, slots, dtype = case["rows"], case["k"], case["n"], case["rank"], case["slots"], DTYPE[case["type"]]
        ids = torch.tensor(rows_slots(case), dtype=torch.int32, device=DEV)
        turn = seed % slots  # another seed gives a request another slot
        ranks = torch.tensor([slot_rank(case, (s - turn) % slots) for s in range(slots)], dtype=torch.int32, device=DEV)
        return {"x": strided(normal(m, k), case["pad"]), "base": strided(normal(m, n), case["pad"]),
                "a": normal(slots, r, k, std=1 / math.sqrt(k)).to(dtype), "b": normal(slots, n, r, std=0.3).to(dtype),
                "ids": torch.where(ids < 0, ids, (ids + turn) % slots), "ranks": ranks,
                "scales": torch.rand(slots, device=DEV, generator=g) + 0.5}
    if case["kind"] == "attn":
        q, o = query_lengths(case), own_lengths(case)
        h, kvh, d, dtype = case["heads"], case["kv_heads"], case["head_dim"], DTYPE[case["type"]]
        capacity = case["own_max"] + 3  # a request's place in the cache of own keys; NaN behind its last one
        table = torch.tensor([sum(q[:i]) for i in range(len(q) + 1)], dtype=torch.int32, device=DEV)
        lens = torch.tensor(o, dtype=torch.int32, device=DEV)
        behind = torch.arange(capacity, device=DEV)[None, :] >= lens[:, None]
        s = {"q": normal(max(1, sum(q)), h * d), "q_start": table, "own_len": lens,
             "own_start": torch.arange(len(o), dtype=torch.int32, device=DEV) * capacity}
        for name in ("k", "v"):
            # keys of one image share a part: scores are not all alike, and some queries peak
            s["prefix_" + name] = normal(case["prefix"], kvh * d, std=1.0 if name == "v" else 0.8, mean=0.3).to(dtype)
            held = normal(len(o), capacity, kvh * d)
            held[behind] = math.nan
            s["own_" + name] = held.view(len(o) * capacity, kvh * d).to(dtype)
        return s
    b, p, c = case["images"], case["pixels"], case["channels"]
    x = normal(b, p, c) * (0.5 + torch.rand(c, device=DEV, generator=g)) + normal(b, 1, c)
    s = {"x": strided(x, case["pad"], DTYPE[case["type"]])}
    if case["affine"]:
        s.update(w=normal(c, std=0.2, mean=1.0), b=normal(c, std=0.2))
    return s


EPS = 1e-5


def prepare(case, seed):
    s = {"case": case, **inputs(case, seed)}
    if own:
        # a program keeps its output buffers and the descriptors of its buffers
        sh, ctx = binding()
        s["ctx"] = ctx
        if case["kind"] == "lora":
            s["y"] = torch.empty(case["rows"], case["n"], device=DEV)
            s["args"] = (sh.lora_bank(describe(sh, s["a"]), describe(sh, s["b"]), s["ranks"].data_ptr(), s["scales"].data_ptr()),
                         describe(sh, s["x"]), sh.tensor(sh.I32, case["rows"], 1, s["ids"].data_ptr()), describe(sh, s["base"]), describe(sh, s["y"]))
        elif case["kind"] == "attn":
            s["y"] = torch.empty_like(s["q"])
            s["args"] = (sh.prefix_attn_desc(
                case["heads"], case["kv_heads"], case["head_dim"], 1 / math.sqrt(case["head_dim"]), describe(sh, s["q"]), describe(sh, s["y"]),
                describe(sh, s["prefix_k"]), describe(sh, s["prefix_v"]), describe(sh, s["own_k"]), describe(sh, s["own_v"]), case["requests"],
                s["q_start"].data_ptr(), s["own_start"].data_ptr(), s["own_len"].data_ptr(), case["own_max"], case["causal"]),)
        else:
            s["y"] = torch.empty(case["images"], case["pixels"], case["channels"], device=DEV, dtype=DTYPE[case["out"]])
            acts = {"none": sh.ACT_NONE, "relu": sh.ACT_RELU, "silu": sh.ACT_SILU, "gelu": sh.ACT_GELU_ERF}
            s["args"] = (describe(sh, s["x"]), describe(sh, s["y"]), case["groups"], s["w"].data_ptr() if "w" in s else None,
                         s["b"].data_ptr() if "b" in s else None, EPS, acts[case["act"]])
        torch.cuda.synchronize()  # the context has a stream of its own
    return s


def describe(sh, t):
    """A ggml descriptor of a torch tensor: dimensions and strides from the innermost."""
    return sh.tensor_nd(sh.F16 if t.dtype == torch.float16 else sh.F32, t.shape[::-1], [v * t.element_size() for v in t.stride()[::-1]], t.data_ptr())


def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "lora":
            s["ctx"].lora_add(*s["args"])
        elif kind == "attn":
            s["ctx"].prefix_attn(*s["args"])
        else:
            s["ctx"].group_norm(*s["args"])
        return s["y"]
    return {"lora": plain_lora, "attn": plain_attn, "norm": plain_norm}[kind](s)


# --- plain forms ---------------------------------------------------------------


def plain_lora(s):
    """Every slot's part of every row, those of other slots and beyond a slot's rank set to zero."""
    a, b, ids = s["a"].float(), s["b"].float(), s["ids"]
    slots, rank, k = a.shape
    t = (s["x"] @ a.view(slots * rank, k).t()).view(-1, slots, rank)
    slot = torch.arange(slots, device=DEV)
    here = (ids[:, None] == slot)[:, :, None] & (torch.arange(rank, device=DEV) < s["ranks"][:, None])
    t = torch.where(here, t * s["scales"][:, None], 0.0)
    return s["base"] + t.view(-1, slots * rank) @ b.permute(0, 2, 1).reshape(slots * rank, -1)


def plain_attn(s):
    case = s["case"]
    h, kvh, d, n_own = case["heads"], case["kv_heads"], case["head_dim"], case["own_max"]
    g, scale, rows, requests = h // kvh, 1 / math.sqrt(d), s["q"].shape[0], case["requests"]
    q = (s["q"] * scale).view(rows, kvh, g, d)
    start, lens = s["q_start"].long(), s["own_len"].long()
    # scores against the prefix, all rows at once
    heads_first = lambda t: t.float().view(-1, kvh, d).permute(1, 2, 0)  # noqa: E731
    pk, pv = heads_first(s["prefix_k"]), heads_first(s["prefix_v"])
    sp = (q.permute(1, 0, 2, 3).reshape(kvh, rows * g, d) @ pk).view(kvh, rows, g, -1)
    # scores against a request's own keys, its queries padded to the longest request's
    slot = torch.arange(case["queries"], device=DEV)
    here = slot < (start[1:] - start[:-1])[:, None]
    place = torch.where(here, start[:-1, None] + slot, 0)
    key = torch.arange(n_own, device=DEV)
    seen = (key < lens[:, None])[:, None, :].expand(requests, case["queries"], n_own)
    if case["causal"]:
        seen = seen & (key <= (lens - (start[1:] - start[:-1]))[:, None, None] + slot[:, None])
    at = (s["own_start"].long()[:, None] + key).clamp(max=s["own_k"].shape[0] - 1)
    real = (key < lens[:, None])[:, :, None]
    ok = torch.where(real, s["own_k"].float()[at], 0.0).view(requests, n_own, kvh, d).permute(0, 2, 3, 1)
    ov = torch.where(real, s["own_v"].float()[at], 0.0).view(requests, n_own, kvh, d).permute(0, 2, 1, 3)
    qp = q[place].permute(0, 2, 1, 3, 4).reshape(requests, kvh, case["queries"] * g, d)
    so = (qp @ ok).view(requests, kvh, case["queries"], g, n_own)
    so = torch.where(seen[:, None, :, None, :], so, -math.inf)
    # back to rows
    row = torch.arange(rows, device=DEV)
    req = (torch.searchsorted(start, row, right=True) - 1).clamp(0, requests - 1)
    pos = (row - start[req]).clamp(0, case["queries"] - 1)
    so = so.permute(0, 2, 1, 3, 4)[req, pos].permute(1, 0, 2, 3)  # kvh, rows, g, own
    most = torch.full((kvh, rows, g, 1), -math.inf, device=DEV)
    if sp.shape[-1]:
        most = torch.maximum(most, sp.amax(-1, keepdim=True))
    if n_own:
        most = torch.maximum(most, so.amax(-1, keepdim=True))
    most = torch.where(torch.isinf(most), 0.0, most)
    sp, so = torch.exp(sp - most), torch.exp(so - most)
    total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    out = (sp.view(kvh, rows * g, -1) @ pv.transpose(1, 2)).view(kvh, rows, g, d)
    wp = torch.zeros(requests, kvh, case["queries"], g, n_own, device=DEV)
    wp = wp.permute(0, 2, 1, 3, 4).index_put((req, pos), so.permute(1, 0, 2, 3)).permute(0, 2, 1, 3, 4)
    op = (wp.reshape(requests, kvh, case["queries"] * g, n_own) @ ov).view(requests, kvh, case["queries"], g, d)
    out = out + op.permute(0, 2, 1, 3, 4)[req, pos].permute(1, 0, 2, 3)
    out = torch.where(total > 0, out / torch.where(total > 0, total, 1.0), 0.0)
    return out.permute(1, 0, 2, 3).reshape(rows, h * d)


def plain_norm(s):
    """Sums in 64 bits: a group of the largest maps has millions of values."""
    case = s["case"]
    x = s["x"].float()
    b, p, c = x.shape
    v = x.reshape(b, p, case["groups"], -1)
    n = v.shape[1] * v.shape[3]
    mean = v.sum((1, 3), keepdim=True, dtype=torch.float64) / n
    centred = v - mean.float()
    var = centred.square().sum((1, 3), keepdim=True, dtype=torch.float64) / n
    y = (centred * (1 / torch.sqrt(var + EPS)).float()).reshape(b, p, c)
    if case["affine"]:
        y = y * s["w"] + s["b"]
    if case["act"] == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif case["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    return y.to(DTYPE[case["out"]])


# --- the definitions in 64 bits ------------------------------------------------


def exact(case, seed):
    s = inputs(case, seed)
    if case["kind"] == "lora":
        y = s["base"].double()
        ids, ranks, scales = s["ids"].tolist(), s["ranks"].tolist(), s["scales"].tolist()
        for slot in sorted(set(ids) - {-1}):
            m, r = (s["ids"] == slot).nonzero()[:, 0], ranks[slot]
            down = s["x"][m].double() @ s["a"][slot, :r].double().t()
            y[m] += scales[slot] * (down @ s["b"][slot, :, :r].double().t())
        return y
    if case["kind"] == "attn":
        h, kvh, d, p = case["heads"], case["kv_heads"], case["head_dim"], case["prefix"]
        start, lens, first = s["q_start"].tolist(), s["own_len"].tolist(), s["own_start"].tolist()
        out = torch.zeros(s["q"].shape[0], h, d, device=DEV, dtype=torch.float64)
        for r in range(case["requests"]):
            n, m = start[r + 1] - start[r], lens[r]
            if not n or not p + m:
                continue
            q = s["q"][start[r]:start[r + 1]].double().view(n, h, d)
            keys, values = (torch.cat([s["prefix_" + x], s["own_" + x][first[r]:first[r] + m]]).double().view(p + m, kvh, d) for x in ("k", "v"))
            hidden = torch.zeros(n, p + m, dtype=torch.bool, device=DEV)
            if case["causal"]:
                i, j = torch.arange(n, device=DEV)[:, None], torch.arange(m, device=DEV)[None, :]
                hidden[:, p:] = j > i + (m - n)
            for head in range(h):
                w = (q[:, head] @ keys[:, head // (h // kvh)].t()) * d ** -0.5
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
                out[start[r]:start[r + 1], head] = w @ values[:, head // (h // kvh)]
        return out.view(-1, h * d)
    x = s["x"].double()
    b, p, c = x.shape
    var, mean = torch.var_mean(x.reshape(b, p, case["groups"], -1), (1, 3), correction=0, keepdim=True)
    y = ((x.reshape(b, p, case["groups"], -1) - mean) * torch.rsqrt(var + EPS)).reshape(b, p, c)
    if case["affine"]:
        y = torch.addcmul(s["b"].double(), y, s["w"].double())
    return {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[case["act"]](y)
