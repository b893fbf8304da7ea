"""A cache of keys and values held in 8 or 4 bits, as cases that can be timed and compared: rotary positions with several axes, K and V rows
rotated and quantised into their requests' pages, rows read back, and attention over such a cache.

`run` computes each in its plain form, or, where `own` is set, by the calls of sam.cpp_amd/samhip.py that a user makes.  Sizes are those
of the repository's benchmark and tests (image tokens 72 x 72, 16 heads of 64 and 8 of 32, 201 queries, 32 or 33 prompt tokens), or generic
ones of the same ranges."""
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

GRID = 72  # image tokens a side


def listed():
    return [
        # One prompt of 32 tokens, all heads of its queries and keys: one launch's latency.
        rope("rotate_32_tokens", 32, 32, 64, "32", "halves", "shared", "f32", "f32"),
        # The queries and keys of an image's tokens in rows of a wider product, an axis for the width and one for the height.
        rope("rotate_image", GRID * GRID, 32, 64, "16,16", "adjacent", "axial", "f32", "f32", pad=1024),
        # Eight frames of image tokens with an axis for time too, some pairs not rotated, F16 in and out.
        rope("rotate_8_frames_f16", 8 * GRID * GRID, 16, 64, "6,12,12", "adjacent", "axial", "f16", "f16"),
        # A token of each of 64 requests into a 4-bit cache: single-token serving, where launches and latency count.
        write("store_64_tokens_q4", 64, 1, 2048, 4, 128, "q4_0", 64, "16,24,24", "halves", "shared", "f16"),
        # Eight prompts of up to 33 tokens behind an image's, small pages, strided rows.
        write("store_8_prompts_q8", 8, 33, 5184 + 33, 8, 32, "q8_0", 16, "16", "halves", "shared", "f32", ragged=True, pad=5),
        # Eight frames of image tokens, rotated in time, height and width, a frame for each request, pages of an odd size.
        write("store_8_frames_q4", 8, GRID * GRID, GRID * GRID, 8, 64, "q4_0", 333, "6,12,12", "adjacent", "axial", "f16"),
        # An image's tokens from an 8-bit cache.
        read("load_image_q8", 1, GRID * GRID, 8, 32, "q8_0", 64, "f32"),
        # Requests of many lengths from a 4-bit cache.
        read("load_24_requests_q4", 24, 8192, 4, 128, "q4_0", 48, "f16"),
        # One query of each of 8 requests on an image's tokens and the request's own.
        attn("attend_single_q4", 8, 1, 5184 + 33, 8, 8, 32, "q4_0", 64),
        # 64 requests, one token each, grouped heads, up to 8192 tokens behind each: long-cache serving.
        attn("attend_64_long_q4", 64, 1, 8192, 16, 4, 128, "q4_0", 64, causal=True),
        # Eight prompts' 201 queries on an image's tokens.
        attn("attend_8_prompts_q8", 8, 201, 5184 + 33, 8, 8, 32, "q8_0", 64),
        # Requests of 0 to 150 queries, causal, with pages that end inside every tile.
        attn("attend_ragged_causal_q8", 13, 150, 1300, 12, 4, 64, "q8_0", 41, causal=True, ragged=True),
    ]


def named(name, c):
    return {"name": name, **c} if name else c


def rope(name, rows, heads, head_dim, pairs, layout, spectrum, type, out, pad=0):
    return named(name, {"kind": "rope", "rows": rows, "heads": heads, "head_dim": head_dim, "pairs": pairs, "layout": layout, "spectrum": spectrum,
                        "type": type, "out": out, "pad": pad})


def write(name, requests, rows, context, kv_heads, head_dim, type, page, pairs, layout, spectrum, out, ragged=False, pad=0):
    return named(name, {"kind": "write", "requests": requests, "queries": rows, "context": context, "kv_heads": kv_heads, "head_dim": head_dim,
                        "type": type, "page": page, "pairs": pairs, "layout": layout, "spectrum": spectrum, "out": out, "causal": True, "ragged": ragged,
                        "pad": pad})


def read(name, requests, context, kv_heads, head_dim, type, page, out, pad=0):
    return named(name, {"kind": "read", "requests": requests, "queries": context, "context": context, "kv_heads": kv_heads, "head_dim": head_dim,
                        "type": type, "page": page, "out": out, "causal": True, "ragged": requests > 1, "pad": pad})


def attn(name, requests, queries, context, heads, kv_heads, head_dim, type, page, causal=False, ragged=False, pad=0):
    return named(name, {"kind": "attn", "requests": requests, "queries": queries, "context": context, "heads": heads, "kv_heads": kv_heads,
                        "head_dim": head_dim, "type": type, "page": page, "causal": causal, "ragged": ragged, "pad": pad})


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _axes(rng, head_dim):
    """One to three axes, most often of all of a head's pairs."""
    half, n = head_dim // 2, rng.randint(1, 3)
    used = half if rng.random() < 0.6 else rng.randint(n, half)
    cuts = sorted(rng.sample(range(1, used), n - 1))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [used]))


def draw(rng):
    kind, head_dim, type = rng.choice(["rope", "write", "read", "attn", "attn"]), rng.choice([32, 64, 128]), rng.choice(["q8_0", "q4_0"])
    layout, spectrum, out = rng.choice(["halves", "adjacent"]), rng.choice(["axial", "shared"]), rng.choice(["f16", "f32"])
    kv_heads, page, pad = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 16, 48, 64, 256, _log(rng, 2, 6000)]), rng.choice([0, 0, 1, 4, 32])
    if kind == "rope":
        heads = rng.randint(1, 40)
        rows = max(1, min(_log(rng, 1, 8 * GRID * GRID), 8 * GRID * GRID * 16 * 64 // (2 * heads * head_dim)))
        return rope(None, rows, heads, head_dim, _axes(rng, head_dim), layout, spectrum, rng.choice(["f16", "f32"]), out, pad)
    width = kv_heads * head_dim
    if kind == "write":
        requests, rows = rng.randint(1, 64), _log(rng, 1, GRID * GRID)
        rows = max(1, min(rows, 8 * GRID * GRID * 512 // (requests * width)))
        context = max(rows, min(_log(rng, 1, 8192), 64 * 8192 * 512 // (requests * width)))
        return write(None, requests, rows, context, kv_heads, head_dim, type, page, _axes(rng, head_dim), layout, spectrum, out, rng.random() < 0.5, pad)
    if kind == "read":
        requests, context = rng.randint(1, 24), _log(rng, 1, 8192)
        return read(None, requests, max(1, min(context, 12 * 8192 * 512 // (requests * width))), kv_heads, head_dim, type, page, out, pad)
    single, group = rng.random() < 0.5, rng.choice([1, 1, 2, 3, 4, 8])
    queries, requests = (1, rng.randint(1, 64)) if single else (_log(rng, 2, 256), rng.randint(1, 12))
    context = max(1, min(_log(rng, 1, 65536), 48 * 8192 * 512 // (requests * width), 8 * 201 * 5184 * 256 // (requests * queries * group * width)))
    return attn(None, requests, queries, context, kv_heads * group, kv_heads, head_dim, type, page, rng.random() < 0.5, not single and rng.random() < 0.7, pad)


# --- what the cases' lengths are (the same for every seed) ---------------------


def spread(i, lo, hi):
    """The i-th of numbers spread over lo .. hi."""
    return lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + 0.37) % 1.0))


def pairs_of(case):
    return [int(v) for v in case["pairs"].split(",")]


def row_counts(case):
    """The rows of each request in the call."""
    if case["kind"] == "read":  # all that it has
        return cache_lengths(case)
    return [spread(r, 0 if r else 1, case["queries"]) if case["ragged"] else case["queries"] for r in range(case["requests"])]


def cache_lengths(case):
    """What each request has in the cache, the call's rows among it."""
    if case["kind"] == "read":
        return [spread(r, 0, case["context"]) if case["ragged"] else case["context"] for r in range(case["requests"])]
    most = case["context"]
    return [max(spread(r, most // 2, most), min(n, most)) for r, n in enumerate(row_counts(case))]


BLOCK_BYTES = {"q8_0": 34, "q4_0": 18}  # of 32 values
THETA = 10000.0


def work(case):
    if case["kind"] == "rope":
        n = case["rows"] * case["heads"] * case["head_dim"]
        turned = 2 * sum(pairs_of(case)) * case["rows"] * case["heads"]
        return {"bytes": n * sum(2 if case[t] == "f16" else 4 for t in ("type", "out")) + 4 * case["rows"] * len(pairs_of(case)), "flops": 3 * turned}
    width, rows, keys = case["kv_heads"] * case["head_dim"], sum(row_counts(case)), sum(cache_lengths(case))
    block = width // 32 * BLOCK_BYTES[case["type"]]
    if case["kind"] == "write":
        return {"bytes": 2 * rows * (4 * width + block + (2 if case["out"] == "f16" else 4) * width), "flops": 8 * rows * width}
    if case["kind"] == "read":
        return {"bytes": 2 * rows * (block + (2 if case["out"] == "f16" else 4) * width), "flops": 2 * rows * width}
    seen = 0
    for n, m in zip(row_counts(case), cache_lengths(case)):
        seen += sum(max(0, m - n + 1 + i) for i in range(n)) if case["causal"] else n * m
    return {"bytes": 8 * rows * case["heads"] * case["head_dim"] + 2 * keys * block, "flops": 4 * seen * case["heads"] * case["head_dim"]}


# --- inputs ------------------------------------------------------------------

DTYPE = {"f32": torch.float32, "f16": torch.float16}


def blocks_q8_0(x):
    """Scales (F16) and codes of 32-value blocks x [..., 32]: d = amax / 127, the codes x * 127 / amax to the nearest, ties to even."""
    amax = x.abs().amax(-1, keepdim=True)
    inverse = torch.where(amax > 0, 127.0 / torch.where(amax > 0, amax, 1.0), 0.0)
    return (amax / 127.0).half(), torch.round(x * inverse).to(torch.int8)


def blocks_q4_0(x):
    """The same in 4 bits: d = m / -8 with m the (first) value of the largest magnitude, the codes x / d + 8 as 0 .. 15."""
    m = x.gather(-1, first_largest(x))
    d = m / -8.0
    inverse = torch.where(d != 0, 1.0 / torch.where(d != 0, d, 1.0), 0.0)
    return d.half(), (x * inverse + 8.5).to(torch.int32).clamp(max=15).to(torch.int8)


def first_largest(x):
    mag = x.abs()
    place = torch.arange(x.shape[-1], device=x.device)
    return torch.where(mag == mag.amax(-1, keepdim=True), place, x.shape[-1]).amin(-1, keepdim=True)


def value_of(d, codes, type):
    return d.float() * (codes.float() - (8.0 if type == "q4_0" else 0.0))


def pack(x, type):
    """Rows [n, width] as cache bytes [n, width / 32 * block bytes]."""
    n = x.shape[0]
    d, codes = (blocks_q8_0 if type == "q8_0" else blocks_q4_0)(x.reshape(n, -1, 32))
    if type == "q4_0":
        codes = codes[..., :16] | (codes[..., 16:] << 4)
    return torch.cat([d.view(torch.uint8), codes.view(torch.uint8)], -1).reshape(n, -1)


def unpack(rows, type):
    """Cache bytes [..., row bytes] as F32 values [..., width]."""
    b = rows.reshape(*rows.shape[:-1], -1, BLOCK_BYTES[type])
    d = b[..., :2].contiguous().view(torch.float16)
    c = b[..., 2:]
    codes = c.contiguous().view(torch.int8) if type == "q8_0" else torch.cat([c & 15, c >> 4], -1)
    return value_of(d, codes, type).flatten(-2)


def inputs(case, seed):
    """Tensors by name, from the seed alone; strided ones hold NaN between their rows, and so do unused rows of a cache."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, device=DEV, generator=g) * std + mean

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    def strided(t, dtype=torch.float32):
        if not case["pad"]:
            return t.to(dtype)
        held = torch.full((t.shape[0], t.shape[1] + case["pad"]), math.nan, device=DEV, dtype=dtype)
        held[:, :t.shape[1]] = t
        return held[:, :t.shape[1]]

    def places(row, position):
        """Positions on one to three axes: a text's, an image's (height, width), a film's (time, height, width)."""
        axes = len(pairs_of(case))
        if axes == 1:
            return position[:, None].contiguous()
        h, w = position // GRID % GRID, position % GRID
        return torch.stack([h, w] if axes == 2 else [position // (GRID * GRID) + row // (GRID * GRID), h, w], 1).contiguous()

    if case["kind"] == "rope":
        row = torch.arange(case["rows"], dtype=torch.int32, device=DEV)
        return {"x": strided(normal(case["rows"], case["heads"] * case["head_dim"]), DTYPE[case["type"]]), "positions": places(row, row + seed % 1000)}
    n, lens, page, width = row_counts(case), cache_lengths(case), case["page"], case["kv_heads"] * case["head_dim"]
    counts = [(m + page - 1) // page for m in lens]
    most, total = max(1, max(counts)), sum(counts) + 1  # a page that nobody has
    order = torch.randperm(total, device=DEV, generator=g).int()
    table = torch.full((len(n), most), -1, dtype=torch.int32, device=DEV)
    for r, c in enumerate(counts):
        table[r, :c] = order[sum(counts[:r]):sum(counts[:r]) + c]
    start = [sum(n[:r]) for r in range(len(n) + 1)]
    rows = start[-1]
    s = {"pages": table, "row_start": ints(start), "len": ints(lens)}
    if case["kind"] == "write":
        s["k"], s["v"] = strided(normal(rows, width, mean=0.2)), strided(normal(rows, width))
        req = torch.repeat_interleave(torch.arange(len(n), device=DEV, dtype=torch.int32), ints(n))
        row = torch.arange(rows, dtype=torch.int32, device=DEV)
        s["positions"] = places(row, row - s["row_start"][req.long()] + ints([m - k for m, k in zip(lens, n)])[req.long()])
        s["cache_rows"] = total * page
        return s
    used = torch.zeros(total * page, dtype=torch.bool, device=DEV)
    for r, m in enumerate(lens):
        at = torch.arange(m, device=DEV)
        used[table[r].long()[at // page] * page + at % page] = True
    for name in "kv":
        # keys of one image share a part: scores are not all alike, and some queries peak
        held = torch.full((total * page, width // 32 * BLOCK_BYTES[case["type"]]), 255, dtype=torch.uint8, device=DEV)
        for at in range(0, total * page, 1 << 16):
            part = normal(min(1 << 16, total * page - at), width, std=1.0 if name == "v" else 0.8, mean=0.3)
            packed = pack(part, case["type"])
            held[at:at + (1 << 16)] = torch.where(used[at:at + (1 << 16), None], packed, 255)
        s[name + "_cache"] = held
    if case["kind"] == "attn":
        s["q"] = strided(normal(rows, case["heads"] * case["head_dim"]))
    return s


def prepare(case, seed):
    s = {"case": case, **inputs(case, seed)}
    if own:
        # a program keeps its output buffers and the descriptors of its buffers
        sh, ctx = binding()
        s["ctx"] = ctx
        turn = None
        if "positions" in s:
            turn = sh.rope_desc(case["head_dim"], pairs_of(case), s["positions"].data_ptr(), sh.ROPE_HALVES if case["layout"] == "halves" else sh.ROPE_ADJACENT,
                                sh.ROPE_SHARED if case["spectrum"] == "shared" else sh.ROPE_AXIAL, THETA)
        if case["kind"] == "rope":
            s["y"] = torch.empty(s["x"].shape, device=DEV, dtype=DTYPE[case["out"]])
            s["args"] = (turn, describe(sh, s["x"]), describe(sh, s["y"]))
        else:
            width, type = case["kv_heads"] * case["head_dim"], {"q8_0": sh.Q8_0, "q4_0": sh.Q4_0}[case["type"]]
            if case["kind"] == "write":
                for name in "kv":
                    s[name + "_cache"] = torch.zeros(s["cache_rows"], width // 32 * BLOCK_BYTES[case["type"]], dtype=torch.uint8, device=DEV)
            k, v = (sh.tensor(type, width, s[name + "_cache"].shape[0], s[name + "_cache"].data_ptr()) for name in "kv")
            cache = sh.kv_cache(case["kv_heads"], case["head_dim"], case["page"], k, v, case["requests"], s["pages"].shape[1], s["pages"].data_ptr(),
                                s["row_start"].data_ptr(), s["len"].data_ptr())
            if case["kind"] == "attn":
                s["y"] = torch.empty(s["q"].shape, device=DEV)
                s["args"] = (sh.cache_attn_desc(case["heads"], case["head_dim"] ** -0.5, cache, describe(sh, s["q"]), describe(sh, s["y"]), case["context"],
                                                case["causal"]),)
            else:
                s["y"] = [torch.empty(sum(row_counts(case)), width, device=DEV, dtype=DTYPE[case["out"]]) for _ in "kv"]
                s["read"] = (cache, *(describe(sh, y) for y in s["y"]))
                if case["kind"] == "write":
                    s["write"] = (cache, turn, describe(sh, s["k"]), describe(sh, s["v"]))
        torch.cuda.synchronize()  # the context has a stream of its own
    return s


def describe(sh, t):
    """A ggml descriptor of a torch tensor: dimensions and strides from the innermost."""
    return sh.tensor_nd(sh.F16 if t.dtype == torch.float16 else sh.F32, t.shape[::-1], [v * t.element_size() for v in t.stride()[::-1]], t.data_ptr())


def run(s):
    """Rows stored in a cache are read back: what is held in a few bits is given as the values it stands for."""
    kind = s["case"]["kind"]
    if own:
        if kind == "rope":
            s["ctx"].rope(*s["args"])
        elif kind == "attn":
            s["ctx"].cache_attn(*s["args"])
        else:
            if kind == "write":
                s["ctx"].cache_write(*s["write"])
            s["ctx"].cache_read(*s["read"])
        return s["y"]
    return {"rope": plain_rope, "write": plain_write, "read": plain_read, "attn": plain_attn}[kind](s)


# --- plain forms ---------------------------------------------------------------


def turned(x, positions, case):
    """Rows [n, heads * head_dim] in F32, each pair of values turned by its axis' position."""
    pairs, hd = pairs_of(case), case["head_dim"]
    total = sum(pairs)
    angle = []  # 64 bits: far positions
    for axis, n in enumerate(pairs):
        j = torch.arange(n, device=DEV, dtype=torch.float64)
        power = j / n if case["spectrum"] == "axial" else (j + sum(pairs[:axis])) / total
        angle.append(positions[:, axis, None].double() * torch.exp(-power * math.log(THETA)))
    angle = torch.cat(angle, 1)[:, None, :]
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    x = x.float().view(x.shape[0], -1, hd)
    first, second = (x[..., 0:2 * total:2], x[..., 1:2 * total:2]) if case["layout"] == "adjacent" else (x[..., :total], x[..., total:2 * total])
    a, b = first * c - second * s, first * s + second * c
    both = torch.stack([a, b], -1).flatten(-2) if case["layout"] == "adjacent" else torch.cat([a, b], -1)
    return torch.cat([both, x[..., 2 * total:]], -1).flatten(1)


def plain_rope(s):
    return turned(s["x"], s["positions"], s["case"]).to(DTYPE[s["case"]["out"]])


def plain_write(s):
    case = s["case"]
    return [unpack(pack(x, case["type"]), case["type"]).to(DTYPE[case["out"]]) for x in (turned(s["k"], s["positions"], case), s["v"])]


def cache_places(s, most):
    """The cache rows of positions 0 .. most - 1 of every request, and which of them are in use."""
    page, at = s["case"]["page"], torch.arange(most, device=DEV)
    real = at < s["len"][:, None]
    return torch.where(real, s["pages"].long()[:, (at // page).clamp(max=s["pages"].shape[1] - 1)] * page + at % page, 0), real


def plain_read(s):
    case = s["case"]
    place, real = cache_places(s, max(cache_lengths(case)))
    return [unpack(s[name][place[real]], case["type"]).to(DTYPE[case["out"]]) for name in ("k_cache", "v_cache")]


def plain_attn(s):
    case = s["case"]
    h, kvh, d, requests = case["heads"], case["kv_heads"], case["head_dim"], case["requests"]
    g, rows, start = h // kvh, s["q"].shape[0], s["row_start"].long()
    most_rows, most_keys = max(1, max(row_counts(case))), max(1, max(cache_lengths(case)))
    place, real = cache_places(s, most_keys)
    k, v = (torch.where(real[..., None], unpack(s[name][place], case["type"]), 0.0).view(requests, most_keys, kvh, d).transpose(1, 2)
            for name in ("k_cache", "v_cache"))
    # each request's queries, padded to the longest request's
    slot, key = torch.arange(most_rows, device=DEV), torch.arange(most_keys, device=DEV)
    n = start[1:] - start[:-1]
    at = torch.where(slot < n[:, None], start[:-1, None] + slot, 0)
    q = (s["q"] * d ** -0.5).view(rows, kvh, g, d)[at].permute(0, 2, 1, 3, 4).reshape(requests, kvh, most_rows * g, d)
    seen = real[:, None, :].expand(requests, most_rows, most_keys)
    if case["causal"]:
        seen = seen & (key <= (s["len"] - n)[:, None, None] + slot[:, None])
    w = (q @ k.transpose(2, 3)).view(requests, kvh, most_rows, g, most_keys)
    w = torch.where(seen[:, None, :, None, :], w, -math.inf)
    most = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(torch.isinf(most), 0.0, most))
    total = w.sum(-1, keepdim=True)
    out = (w.view(requests, kvh, most_rows * g, most_keys) @ v).view(requests, kvh, most_rows, g, d)
    out = torch.where(total > 0, out / torch.where(total > 0, total, 1.0), 0.0)
    # back to rows
    row = torch.arange(rows, device=DEV)
    req = (torch.searchsorted(start, row, right=True) - 1).clamp(0, requests - 1)
    return out[req, :, (row - start[req]).clamp(0, most_rows - 1)].reshape(rows, h * d)


# --- the definitions in 64 bits ------------------------------------------------


def exact_rows(x, positions, case):
    """The rotation with cos and sin as F32 numbers, the rest in 64 bits."""
    pairs, hd = pairs_of(case), case["head_dim"]
    y = x.double().view(x.shape[0], -1, hd).clone()
    p = 0
    for axis, n in enumerate(pairs):
        for j in range(n):
            frequency = THETA ** (-j / n if case["spectrum"] == "axial" else -p / sum(pairs))
            angle = positions[:, axis].double() * frequency
            c, s = (f(angle).float().double()[:, None] for f in (torch.cos, torch.sin))
            a, b = (2 * p, 2 * p + 1) if case["layout"] == "adjacent" else (p, p + sum(pairs))
            u, v = y[:, :, a].clone(), y[:, :, b].clone()
            if case["kind"] == "write":  # what is quantised is an F32 number: each product and their sum rounded
                y[:, :, a] = ((u * c).float().double() - (v * s).float().double()).float().double()
                y[:, :, b] = ((u * s).float().double() + (v * c).float().double()).float().double()
            else:
                y[:, :, a], y[:, :, b] = u * c - v * s, u * s + v * c
            p += 1
    return y.view(x.shape)


def exact_stored(x, type):
    """What a block of 32 holds of F32 values given in 64 bits; the scale and its inverse are F32 numbers, the stored scale F16."""
    x = x.reshape(x.shape[0], -1, 32)
    r = lambda t: t.float().double()  # noqa: E731
    if type == "q8_0":
        amax = x.abs().max(-1, keepdim=True).values
        codes = torch.round(r(x * r(127.0 / amax).nan_to_num(posinf=0.0)))
        return (r(amax / 127.0).half().double() * codes).flatten(1)
    hi, lo = x.max(-1, keepdim=True).values, x.min(-1, keepdim=True).values
    d = torch.where(hi > -lo, hi, torch.where(hi < -lo, lo, x.gather(-1, first_largest(x)))) / -8.0
    codes = torch.floor(r(r(x * r(1.0 / d).nan_to_num(posinf=0.0, neginf=0.0)) + 8.5)).clamp(max=15.0)
    return (d.half().double() * (codes - 8.0)).flatten(1)


def exact_loaded(rows, type):
    """Cache bytes as values in 64 bits."""
    b = rows.reshape(rows.shape[0], rows.shape[1] // BLOCK_BYTES[type], BLOCK_BYTES[type])
    d = (b[:, :, 0].short() | (b[:, :, 1].short() << 8)).view(torch.float16).double()[..., None]
    c = b[:, :, 2:].double()
    if type == "q8_0":
        return (d * torch.where(c > 127, c - 256, c)).flatten(1)
    high = torch.floor(c / 16)
    return (d * (torch.cat([c - 16 * high, high], -1) - 8)).flatten(1)


def exact(case, seed):
    s = inputs(case, seed)
    if case["kind"] == "rope":
        return exact_rows(s["x"], s["positions"], case)
    if case["kind"] == "write":
        return [exact_stored(x, case["type"]) for x in (exact_rows(s["k"], s["positions"], case), s["v"].double())]
    start, lens, page, d = s["row_start"].tolist(), s["len"].tolist(), case["page"], case["head_dim"]
    at = [s["pages"][r].long().repeat_interleave(page)[:m] * page + torch.arange(m, device=DEV) % page for r, m in enumerate(lens)]
    if case["kind"] == "read":
        return [torch.cat([exact_loaded(s[name][rows], case["type"]) for rows in at]) for name in ("k_cache", "v_cache")]
    h, kvh = case["heads"], case["kv_heads"]
    out = torch.zeros(s["q"].shape[0], h, d, device=DEV, dtype=torch.float64)
    for r, m in enumerate(lens):
        n = start[r + 1] - start[r]
        if not n or not m:
            continue
        keys, values = (exact_loaded(s[name][at[r]], case["type"]).view(m, kvh, d) for name in ("k_cache", "v_cache"))
        q = s["q"][start[r]:start[r + 1]].double().view(n, h, d)
        hidden = torch.zeros(n, m, dtype=torch.bool, device=DEV)
        if case["causal"]:
            hidden = torch.arange(m, device=DEV)[None, :] > torch.arange(n, device=DEV)[:, None] + (m - n)
        for head in range(h):
            w = (q[:, head] @ keys[:, head // (h // kvh)].t()) * d ** -0.5
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
            out[start[r]:start[r + 1], head] = w @ values[:, head // (h // kvh)]
    return out.view(-1, h * d)
