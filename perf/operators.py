"""Operators of a decode loop over forked and prefix-cached requests, measured against plain torch forms.

Three operators over one paged cache (K and V of [pages][kv_heads][16][head_size]):

* ``shared``: batch decode attention in which groups of consecutive rows share their leading pages;
* ``pages`` / ``slots``: whole pages, or single tokens' rows, copied inside the caches of all layers at once;
* ``rotate``: per-head RMS norm of Q and K, rotary positions, and the write of K and V into their cache slots.

With ``own`` set, ``run`` calls the framework; without it, elementary torch operations in 32 bits.
"""
import ctypes
import math

import torch

own = False

BS = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # Four samples of one short prompt on a small model: a call that is all latency.
        {"name": "shared_small", "op": "shared", "dtype": "bf16", "groups": 1, "rows": 4, "q_heads": 8, "kv_heads": 2, "hd": 128,
         "prefix_min": 512, "prefix_max": 512, "suffix_min": 1, "suffix_max": 32},
        # Sixteen samples of one prompt, fp16, head size 64, ragged answers.
        {"name": "shared_sampling_f16", "op": "shared", "dtype": "f16", "groups": 1, "rows": 16, "q_heads": 32, "kv_heads": 8, "hd": 64,
         "prefix_min": 2064, "prefix_max": 2064, "suffix_min": 1, "suffix_max": 500},
        # Eight system prompts of different lengths, eight conversations behind each.
        {"name": "shared_prompts", "op": "shared", "dtype": "bf16", "groups": 8, "rows": 8, "q_heads": 32, "kv_heads": 8, "hd": 128,
         "prefix_min": 1024, "prefix_max": 8192, "suffix_min": 16, "suffix_max": 1024},
        # Sixty-four short questions about one long document.
        {"name": "shared_document", "op": "shared", "dtype": "f16", "groups": 1, "rows": 64, "q_heads": 32, "kv_heads": 8, "hd": 128,
         "prefix_min": 32768, "prefix_max": 32768, "suffix_min": 16, "suffix_max": 300},
        # A full batch behind one long prompt, with long conversations of their own.
        {"name": "shared_full_batch", "op": "shared", "dtype": "bf16", "groups": 1, "rows": 256, "q_heads": 64, "kv_heads": 8, "hd": 128,
         "prefix_min": 16384, "prefix_max": 16384, "suffix_min": 200, "suffix_max": 2000},
        # One request forked eight ways: its partial last page, one layer.
        {"name": "pages_fork", "op": "pages", "dtype": "bf16", "layers": 1, "pool": 512, "kv_heads": 8, "hd": 128, "count": 8, "fanout": 8},
        # A batch of forks over all layers of a model.
        {"name": "pages_layers", "op": "pages", "dtype": "bf16", "layers": 32, "pool": 512, "kv_heads": 8, "hd": 128, "count": 96, "fanout": 4},
        # Eviction keeps about half of an fp32 sequence's tokens, odd counts.
        {"name": "slots_f32", "op": "slots", "dtype": "f32", "layers": 4, "pool": 512, "kv_heads": 2, "hd": 64, "count": 1111, "length": 2345},
        # Eviction in a long sequence of a 16-layer model.
        {"name": "slots_layers", "op": "slots", "dtype": "bf16", "layers": 16, "pool": 1600, "kv_heads": 8, "hd": 128, "count": 8190,
         "length": 16380},
        # One decode step's new tokens.
        {"name": "rotate_decode", "op": "rotate", "dtype": "bf16", "tokens": 64, "q_heads": 32, "kv_heads": 8, "hd": 128, "rotary": 128,
         "interleaved": False, "norm": True, "pool": 1024},
        # An odd prefill chunk, fp16, head size 64, half of each head rotated in adjacent pairs.
        {"name": "rotate_partial_f16", "op": "rotate", "dtype": "f16", "tokens": 777, "q_heads": 16, "kv_heads": 2, "hd": 64, "rotary": 32,
         "interleaved": True, "norm": True, "pool": 1024},
        # A large prefill chunk.
        {"name": "rotate_prefill", "op": "rotate", "dtype": "bf16", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "hd": 128, "rotary": 128,
         "interleaved": False, "norm": True, "pool": 1024},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["shared", "shared", "pages", "slots", "rotate"])
    if op == "shared":
        hd, kv_heads, group = rng.choice([64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12])
        groups = _log(rng, 1, 12)
        rows = _log(rng, 1, 256 // groups)
        # No more prefix work, and no more suffix bytes, than the largest listed case.
        most = 16384 * 256 * 64 // (groups * rows * kv_heads * group)
        prefix_max = max(1, min(_log(rng, 1, 2048), most // 16, 65536 // groups // 16)) * 16
        suffix_max = max(1, min(_log(rng, 1, 2000), 256 * 2000 // (groups * rows)))
        return {"op": op, "dtype": rng.choice(["bf16", "f16"]), "groups": groups, "rows": rows, "q_heads": kv_heads * group, "kv_heads": kv_heads,
                "hd": hd, "prefix_min": max(16, prefix_max // 2 // 16 * 16), "prefix_max": prefix_max,
                "suffix_min": rng.choice([0, 1, max(1, suffix_max // 3)]), "suffix_max": suffix_max}
    dtype, hd, kv_heads, layers = rng.choice(["bf16", "f16", "f32"]), rng.choice([32, 64, 128, 256]), rng.choice([1, 2, 4, 8]), _log(rng, 1, 16)
    if op == "pages":
        count = _log(rng, 1, 128)
        return {"op": op, "dtype": dtype, "layers": layers, "pool": 300, "kv_heads": kv_heads, "hd": hd, "count": count, "fanout": rng.choice([1, 1, 2, 5, 16])}
    if op == "slots":
        length = _log(rng, 2, 2500)
        return {"op": op, "dtype": dtype, "layers": layers, "pool": 400, "kv_heads": kv_heads, "hd": hd, "count": rng.randint(1, length), "length": length}
    return {"op": op, "dtype": dtype, "tokens": _log(rng, 1, 4000), "q_heads": kv_heads * rng.choice([1, 2, 4, 5, 8]), "kv_heads": kv_heads,
            "hd": hd, "rotary": rng.choice([hd, hd, hd // 2]), "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.8, "pool": 512}


# ---------------------------------------------------------------- inputs ---

def _ints(gen, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=gen)


def _values(seed, shape, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype)


def prepare(case, seed):
    return {"shared": _prepare_shared, "pages": _prepare_pages, "slots": _prepare_slots, "rotate": _prepare_rotate}[case["op"]](case, seed)


def _prepare_shared(case, seed):
    gen = torch.Generator().manual_seed(seed)
    groups, rows, hq, hkv, hd = case["groups"], case["rows"], case["q_heads"], case["kv_heads"], case["hd"]
    batch, dt = groups * rows, DTYPES[case["dtype"]]
    prefix = _ints(gen, case["prefix_min"] // BS, case["prefix_max"] // BS, groups) * BS
    suffix = _ints(gen, case["suffix_min"], case["suffix_max"], batch)
    lens = prefix.repeat_interleave(rows) + suffix
    pages_p, pages_s = case["prefix_max"] // BS, -(-case["suffix_max"] // BS)
    width = pages_p + pages_s
    # The pool's pages in a random order: the groups' prefixes first, then each row's own pages; -1 past a row's end.
    num_pages = groups * pages_p + batch * pages_s
    ids = torch.randperm(num_pages, generator=gen)
    shared_ids = ids[:groups * pages_p].view(groups, pages_p).repeat_interleave(rows, 0)
    own_ids = ids[groups * pages_p:].view(batch, pages_s)
    col = torch.arange(width).expand(batch, width)
    start = (prefix // BS).repeat_interleave(rows)[:, None]
    table = torch.where(col < start, shared_ids.gather(1, col.clamp(max=pages_p - 1)), own_ids.gather(1, (col - start).clamp(0, pages_s - 1)))
    table = torch.where(col < (lens[:, None] + BS - 1) // BS, table, torch.full_like(table, -1))
    shape = (num_pages, hkv, BS, hd)
    return {"case": case, "q": _values(seed * 4 + 1, (batch, hq, hd), torch.float32), "o": torch.zeros(batch, hq, hd, device="cuda"),
            "k": _values(seed * 4 + 2, shape, dt), "v": _values(seed * 4 + 3, shape, dt), "table": table.contiguous().cuda(), "lens": lens.cuda(),
            "prefix": prefix.cuda(), "prefix_host": prefix.tolist(), "max_len": width * BS}


def _prepare_pages(case, seed):
    gen = torch.Generator().manual_seed(seed)
    n, pool = case["count"], case["pool"]
    ids = torch.randperm(pool, generator=gen)
    sources = ids[:-(-n // case["fanout"])].repeat_interleave(case["fanout"])[:n]
    kv = _values(seed * 4 + 1, (case["layers"], 2, pool, case["kv_heads"], BS, case["hd"]), DTYPES[case["dtype"]])
    return {"case": case, "kv": kv, "src": sources.contiguous().cuda(), "dst": ids[pool - n:].contiguous().cuda()}


def _prepare_slots(case, seed):
    gen = torch.Generator().manual_seed(seed)
    n, length, pool = case["count"], case["length"], case["pool"]
    ids = torch.randperm(pool, generator=gen)
    keep = torch.randperm(length, generator=gen)[:n].sort().values
    at = torch.arange(n)
    fresh = ids[-(-length // BS):]
    kv = _values(seed * 4 + 1, (case["layers"], 2, pool, case["kv_heads"], BS, case["hd"]), DTYPES[case["dtype"]])
    return {"case": case, "kv": kv, "src": (ids[keep // BS] * BS + keep % BS).cuda(), "dst": (fresh[at // BS] * BS + at % BS).cuda()}


def _prepare_rotate(case, seed):
    gen = torch.Generator().manual_seed(seed)
    n, hq, hkv, hd, rot = case["tokens"], case["q_heads"], case["kv_heads"], case["hd"], case["rotary"]
    dt, reach = DTYPES[case["dtype"]], 32768
    angle = torch.arange(reach, dtype=torch.float64, device="cuda")[:, None] * \
        torch.pow(10000.0, -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    cache = (case["pool"], hkv, BS, hd)
    state = {"case": case, "qkv": _values(seed * 4 + 1, (n, hq + 2 * hkv, hd), dt), "k": _values(seed * 4 + 2, cache, dt),
             "v": _values(seed * 4 + 3, cache, dt), "q_out": torch.zeros(n, hq, hd, device="cuda"),
             "cos_sin": torch.cat([angle.cos(), angle.sin()], 1).float().contiguous(), "eps": 1e-6,
             "positions": _ints(gen, 0, reach - 1, n).cuda(), "slots": torch.randperm(case["pool"] * BS, generator=gen)[:n].cuda()}
    if case["norm"]:
        state["q_weight"] = 1 + 0.1 * _values(seed * 4 + 4, (hd,), torch.float32)
        state["k_weight"] = 1 + 0.1 * _values(seed * 4 + 5, (hd,), torch.float32)
    return state


# ------------------------------------------------------------------ runs ---

def run(state):
    op = state["case"]["op"]
    if own:
        return {"shared": _own_shared, "pages": _own_copy, "slots": _own_copy, "rotate": _own_rotate}[op](state)
    return {"shared": _plain_shared, "pages": _plain_pages, "slots": _plain_slots, "rotate": _plain_rotate}[op](state)


def _plain_shared(s):
    c = s["case"]
    groups, rows, hkv, hd = c["groups"], c["rows"], c["kv_heads"], c["hd"]
    batch, g = groups * rows, c["q_heads"] // c["kv_heads"]
    pages_p, width = c["prefix_max"] // BS, s["table"].shape[1]
    q = s["q"].view(batch, hkv, g, hd) / math.sqrt(hd)
    # The groups' prefixes, read once through their first rows' tables.
    ids = s["table"].view(groups, rows, width)[:, 0, :pages_p].clamp(min=0)
    kp = s["k"][ids].float().transpose(2, 3).reshape(groups, pages_p * BS, hkv, hd)
    vp = s["v"][ids].float().transpose(2, 3).reshape(groups, pages_p * BS, hkv, hd)
    sp = torch.einsum("grhqd,gphd->grhqp", q.view(groups, rows, hkv, g, hd), kp)
    dead = torch.arange(pages_p * BS, device=q.device) >= s["prefix"][:, None]
    sp = sp.masked_fill(dead[:, None, None, None, :], -math.inf).reshape(batch, hkv, g, -1)
    # The rows' own tokens.
    pages_s = width - pages_p
    first = s["prefix"].repeat_interleave(rows)
    cols = ((first // BS)[:, None] + torch.arange(pages_s, device=q.device)).clamp(max=width - 1)
    ids = s["table"].gather(1, cols).clamp(min=0)
    ks = s["k"][ids].float().transpose(2, 3).reshape(batch, pages_s * BS, hkv, hd)
    vs = s["v"][ids].float().transpose(2, 3).reshape(batch, pages_s * BS, hkv, hd)
    ss = torch.einsum("bhqd,bshd->bhqs", q, ks)
    dead = torch.arange(pages_s * BS, device=q.device) >= (s["lens"] - first)[:, None]
    ss = ss.masked_fill(dead[:, None, None, :], -math.inf)
    top = torch.maximum(sp.amax(-1), ss.amax(-1))[..., None]
    pp, ps = torch.exp(sp - top), torch.exp(ss - top)
    o = torch.einsum("grhqp,gphd->grhqd", pp.reshape(groups, rows, hkv, g, -1), vp).reshape(batch, hkv, g, hd)
    o = (o + torch.einsum("bhqs,bshd->bhqd", ps, vs)) / (pp.sum(-1) + ps.sum(-1))[..., None]
    s["o"].copy_(o.reshape(batch, hkv * g, hd))
    return s["o"]


def _plain_pages(s):
    s["kv"][:, :, s["dst"]] = s["kv"][:, :, s["src"]]
    return s["kv"]


def _plain_slots(s):
    kv, src, dst = s["kv"], s["src"], s["dst"]
    kv[:, :, dst // BS, :, dst % BS] = kv[:, :, src // BS, :, src % BS]
    return kv


def _plain_rotate(s):
    c = s["case"]
    hq, hkv, rot = c["q_heads"], c["kv_heads"], c["rotary"]
    q, k, v = s["qkv"].split([hq, hkv, hkv], 1)
    x, y = q.float(), k.float()
    if c["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * s["q_weight"]
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * s["k_weight"]
    cos, sin = s["cos_sin"][s["positions"]][:, None].split(rot // 2, 2)
    x, y = _plain_turn(x, cos, sin, c), _plain_turn(y, cos, sin, c)
    s["q_out"].copy_(x)
    page, off = s["slots"] // BS, s["slots"] % BS
    s["k"][page, :, off] = y.to(s["k"].dtype)
    s["v"][page, :, off] = v
    return s["q_out"], s["k"], s["v"]


def _plain_turn(x, cos, sin, c):
    rot = c["rotary"]
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _cache(kv, k, v, case):
    # K and V as [pages][kv_heads][BS][head_size].
    return kv.KvfxCache(k.data_ptr(), v.data_ptr(), k.shape[0], k.shape[1], k.shape[2], k.shape[3],
                        {"f16": kv.KVFX_F16, "bf16": kv.KVFX_BF16, "f32": kv.KVFX_F32}[case["dtype"]], k.device.index, 0)


def _own_shared(s):
    import kvflux_b200 as kv

    c = s["case"]
    if "plan" not in s:  # what a serving loop keeps from step to step: descriptor, groups, workspace
        cache = _cache(kv, s["k"], s["v"], c)
        groups = (kv.KvfxPrefixGroup * c["groups"])(*[(c["rows"], p) for p in s["prefix_host"]])
        need = kv.lib.kvfx_decode_shared_workspace_bytes(ctypes.byref(cache), groups, c["groups"], c["q_heads"], s["max_len"])
        s["plan"] = cache, groups, need, torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    cache, groups, need, ws = s["plan"]
    kv.check(kv.lib.kvfx_decode_shared(ctypes.byref(cache), s["q"].data_ptr(), s["o"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(),
                                       groups, c["groups"], s["table"].shape[1], c["q_heads"], s["max_len"], ws.data_ptr(), need, _stream()),
             "kvfx_decode_shared")
    return s["o"]


def _own_copy(s):
    import kvflux_b200 as kv

    if "plan" not in s:
        s["plan"] = (kv.KvfxCache * s["case"]["layers"])(*[_cache(kv, layer[0], layer[1], s["case"]) for layer in s["kv"]])
    call = kv.lib.kvfx_copy_pages if s["case"]["op"] == "pages" else kv.lib.kvfx_copy_slots
    kv.check(call(s["plan"], s["case"]["layers"], s["src"].data_ptr(), s["dst"].data_ptr(), s["src"].numel(), _stream()), "kvfx_copy")
    return s["kv"]


def _own_rotate(s):
    import kvflux_b200 as kv

    c = s["case"]
    hq, hkv, hd = c["q_heads"], c["kv_heads"], c["hd"]
    if "plan" not in s:
        weights = [s[w].data_ptr() if c["norm"] else None for w in ("q_weight", "k_weight")]
        s["plan"] = (_cache(kv, s["k"], s["v"], c),
                     kv.KvfxRotary(s["cos_sin"].data_ptr(), s["cos_sin"].shape[0], c["rotary"], int(c["interleaved"]), *weights, s["eps"], 0))
    cache, rotary = s["plan"]
    q, step, row = s["qkv"].data_ptr(), (hq + 2 * hkv) * hd, hd * s["qkv"].element_size()
    kv.check(kv.lib.kvfx_write_rotated(ctypes.byref(cache), ctypes.byref(rotary), q, q + hq * row, q + (hq + hkv) * row, step, step, step, hq,
                                       s["positions"].data_ptr(), s["slots"].data_ptr(), c["tokens"], s["q_out"].data_ptr(), _stream()),
             "kvfx_write_rotated")
    return s["q_out"], s["k"], s["v"]


# ------------------------------------------------------- work and 64 bits ---

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "shared":
        row = 2 * case["kv_heads"] * case["hd"] * e
        prefix = (case["prefix_min"] + case["prefix_max"]) // 2
        suffix = (case["suffix_min"] + case["suffix_max"]) / 2
        batch = case["groups"] * case["rows"]
        io = 2 * batch * case["q_heads"] * case["hd"] * 4
        table = 8 * (case["groups"] * prefix // BS + batch * -(-suffix // BS) + batch)
        return {"bytes": case["groups"] * prefix * row + batch * suffix * row + io + table,
                "flops": 4.0 * batch * (prefix + suffix) * case["q_heads"] * case["hd"]}
    if case["op"] in ("pages", "slots"):
        row = 2 * case["kv_heads"] * case["hd"] * e * case["layers"] * (BS if case["op"] == "pages" else 1)
        read = -(-case["count"] // case.get("fanout", 1))
        return {"bytes": (read + case["count"]) * row + 16 * case["count"], "flops": 0}
    heads = case["q_heads"] + 2 * case["kv_heads"]
    n, hd = case["tokens"], case["hd"]
    return {"bytes": n * hd * (heads * e + case["q_heads"] * 4 + 2 * case["kv_heads"] * e) + n * (case["rotary"] * 4 + 16),
            "flops": n * hd * (case["q_heads"] + case["kv_heads"]) * 9.0}


def exact(case, seed):
    if case["op"] in ("pages", "slots"):
        return None  # moved, not computed
    return _exact_shared(case, seed) if case["op"] == "shared" else _exact_rotate(case, seed)


def _exact_shared(case, seed):
    s = _prepare_shared(case, seed)
    hkv, hd = case["kv_heads"], case["hd"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    for r, length in enumerate(s["lens"].tolist()):
        # Every position of the row through its own table, one softmax over all of them.
        t = torch.arange(length, device="cuda")
        page, off = s["table"][r][t // BS], t % BS
        key, value = (s[w][page, :, off].double().permute(1, 0, 2) for w in ("k", "v"))
        q = s["q"][r].double().view(hkv, -1, hd)
        weight = torch.softmax(torch.bmm(q, key.transpose(1, 2)) * hd ** -0.5, dim=-1)
        out[r] = torch.bmm(weight, value).reshape(-1, hd)
    return out


def _exact_rotate(case, seed):
    s = _prepare_rotate(case, seed)
    hq, hkv, rot, half = case["q_heads"], case["kv_heads"], case["rotary"], case["rotary"] // 2
    x = s["qkv"].double()
    if case["norm"]:
        scale = (x.square().sum(-1) / case["hd"] + s["eps"]).sqrt()
        weight = torch.stack([s["q_weight"]] * hq + [s["k_weight"]] * hkv).double()
        x = torch.cat([x[:, :hq + hkv] / scale[:, :hq + hkv, None] * weight, x[:, hq + hkv:]], 1)
    # Each pair as a complex number, turned by the unit number of its angle.
    table = s["cos_sin"].double()[s["positions"]]
    unit = torch.complex(table[:, :half], table[:, half:])[:, None]
    first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    turned = torch.complex(x[:, :hq + hkv, first], x[:, :hq + hkv, second]) * unit
    y = x.clone()
    y[:, :hq + hkv, first], y[:, :hq + hkv, second] = turned.real, turned.imag
    k, v = s["k"].double(), s["v"].double()
    for i, slot in enumerate(s["slots"].tolist()):
        k[slot // BS, :, slot % BS] = y[i, hq:hq + hkv]
        v[slot // BS, :, slot % BS] = y[i, hq + hkv:]
    return y[:, :hq].contiguous(), k, v
