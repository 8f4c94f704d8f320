"""What the 8-bit KV cache of this library and the operators around it are measured on.

One layer's calls of a serving step: rotary positions, the append of new keys and values to pages that hold 8 bits a value
and one scale per page and KV head, attention over those pages, and eviction by accumulated attention weight.

Layouts: q ``[tokens, hq, d]``, k and v ``[tokens, hkv, d]``; cache pages ``[pages, hkv, page, d]`` of int8 or e4m3 with
scales ``[pages, hkv]`` and accumulated weights ``[pages, hkv, page]``; a sequence is a row of the page table, its length
(this step's new tokens included) and the run of rows of q, k and v that its new tokens are.  Values: q, k, v ~ N(0, 1), some
channels of k four times as large, as rotary models have them; the cache holds such values quantised.
"""
import math
import random

import torch

own = False

TOP = {"int8": 127.0, "e4m3": 448.0}    # the largest value of the 8-bit types
CACHE_TYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
IO_TYPE = {"fp16": torch.float16, "bf16": torch.bfloat16}
BASE = 10000.0


# ---- cases --------------------------------------------------------------------------------------------------------

def _rotary(tokens, hq, hkv, d, part, layout, scaling, far, dtype, name=None):
    c = {"op": "rotary", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "part": part, "layout": layout,
         "scaling": scaling, "far": far, "dtype": dtype}
    return c if name is None else {**c, "name": name}


def _append(seqs, old, new, hq, hkv, d, page, kind, layout, dtype, name=None):
    """old, new: texts like "0-4096": the lengths of the cached part and of the new part of the sequences."""
    c = {"op": "append", "seqs": seqs, "old": old, "new": new, "hq": hq, "hkv": hkv, "d": d, "page": page,
         "kind": kind, "layout": layout, "dtype": dtype}
    return c if name is None else {**c, "name": name}


def _attend(seqs, old, new, hq, hkv, d, page, kind, window, weights, dtype, name=None):
    c = {"op": "attend", "seqs": seqs, "old": old, "new": new, "hq": hq, "hkv": hkv, "d": d, "page": page,
         "kind": kind, "window": window, "weights": weights, "dtype": dtype}
    return c if name is None else {**c, "name": name}


def _evict(seqs, old, budget, recent, hkv, d, page, kind, dtype, name=None):
    c = {"op": "evict", "seqs": seqs, "old": old, "new": "0-0", "budget": budget, "recent": recent, "hkv": hkv, "d": d,
         "page": page, "kind": kind, "dtype": dtype}
    return c if name is None else {**c, "name": name}


def listed():
    return [
        # a decode step of a lone request: launch and latency are all there is
        _rotary(1, 32, 32, 128, 128, "half", "none", 4000, "fp16", "rotary_one_token"),
        # a long prompt of a model that rotates half of each head in pairs of neighbours, scaled for 128k positions
        _rotary(8191, 64, 8, 128, 64, "interleaved", "yarn", 131000, "bf16", "rotary_prompt_yarn"),
        # one new token for each of 77 requests, 7B-shaped: rotated, quantised, some pages rescaled
        _append(77, "1-4000", "1-1", 32, 32, 128, 16, "int8", "half", "fp16", "append_decode_7b"),
        # prompts of any length into empty and half-filled pages, grouped heads, e4m3
        _append(9, "0-100", "300-2048", 64, 8, 128, 64, "e4m3", "half", "bf16", "append_prompts_gqa"),
        # the smallest attention: one request with a short context
        _attend(1, "128-128", "1-1", 32, 32, 128, 16, "int8", 0, False, "fp16", "attend_one_short"),
        # the decode step of a 7B-shaped model: every head has keys of its own, lengths ragged
        _attend(64, "64-4096", "1-1", 32, 32, 128, 16, "int8", 0, False, "fp16", "attend_decode_7b"),
        # few requests with very long contexts, eight query heads to a KV head (the 70B shape)
        _attend(16, "8192-65536", "1-1", 64, 8, 128, 64, "int8", 0, False, "bf16", "attend_decode_gqa_long"),
        # decode that also gathers the attention weight of every cached token, which eviction goes by
        _attend(32, "1000-8192", "1-1", 32, 8, 128, 32, "e4m3", 0, True, "bf16", "attend_decode_weights"),
        # a few drafted tokens of each request checked at once, sliding window
        _attend(24, "500-8000", "2-5", 64, 8, 128, 32, "int8", 4096, False, "fp16", "attend_verify_window"),
        # chunks of long prompts over what is cached of them
        _attend(4, "1000-6000", "512-2048", 64, 8, 128, 64, "int8", 0, False, "bf16", "attend_chunks_gqa"),
        # a few sequences brought back to 512 tokens
        _evict(4, "1000-2000", 512, 128, 8, 128, 16, "int8", "fp16", "evict_few"),
        # a batch of long sequences brought back to 2048 tokens
        _evict(32, "3000-16000", 2048, 512, 8, 128, 32, "int8", "bf16", "evict_many"),
    ]


def _spread(rng, lo, hi):
    """Uniform over the logarithm, odd sizes included."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "attend", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    kind = rng.choice(["int8", "int8", "e4m3"])
    page = rng.choice([16, 32, 64])
    d = rng.choice([64, 128, 128])
    hq, hkv = rng.choice([(32, 32), (40, 40), (32, 8), (64, 8), (40, 8), (16, 1)])
    if op == "rotary":
        part = rng.choice([d, d, d // 2, d // 4])
        return _rotary(_spread(rng, 1, 8000), hq, hkv, d, part, rng.choice(["half", "interleaved"]),
                       rng.choice(["none", "linear", "ntk", "yarn", "llama3"]), _spread(rng, 2000, 200000), dtype)
    if op == "append":
        if rng.random() < 0.5:
            return _append(_spread(rng, 1, 256), "0-%d" % _spread(rng, 1, 4000), "1-1", hq, hkv, d, page, kind,
                           rng.choice(["half", "interleaved"]), dtype)
        return _append(_spread(rng, 1, 16), "0-%d" % _spread(rng, 1, 500), "1-%d" % _spread(rng, 2, 1024), hq, hkv, d, page,
                       kind, rng.choice(["half", "interleaved"]), dtype)
    if op == "evict":
        budget = _spread(rng, 64, 2048)
        top = _spread(rng, budget + 1, 16000)
        return _evict(_spread(rng, 1, 24), "%d-%d" % (max(1, budget // 2), top), budget,
                      rng.randrange(0, budget // 2), min(hkv, 8), d, page, kind, dtype)
    form = rng.random()
    if form < 0.6:
        seqs, new = _spread(rng, 1, 128), "1-1"
    elif form < 0.8:
        seqs, new = _spread(rng, 1, 32), "1-%d" % _spread(rng, 2, 8)
    else:
        seqs, new = _spread(rng, 1, 4), "16-%d" % _spread(rng, 64, 1024)
    longest = int(new.split("-")[1])
    top = min(_spread(rng, 16, 65536), 2 ** 21 // (seqs * hkv), 2 ** 32 // (seqs * hq * longest) - longest)
    window = rng.choice([0, 0, 0, _spread(rng, 16, 8192)])
    weights = rng.random() < 0.25
    return _attend(seqs, "%d-%d" % (max(0, top // rng.choice([1, 4, 16]) - 1), top), new, hq, hkv, d, page, kind, window, weights,
                   dtype)


def _lengths(case):
    """Cached and new tokens of each sequence: they belong to the case, the values to the seed."""
    rng = random.Random("%s %s %s" % (case["seqs"], case["old"], case["new"]))
    (a, b), (c, e) = ([int(x) for x in case[k].split("-")] for k in ("old", "new"))
    old = [_spread(rng, max(1, a), max(1, b)) if b else 0 for _ in range(case["seqs"])]
    if a == 0:
        old = [x if rng.random() < 0.7 else 0 for x in old]
    return old, [_spread(rng, c, e) if e else 0 for _ in range(case["seqs"])]


def work(case):
    if case["op"] == "rotary":
        n = case["tokens"] * (case["hq"] + case["hkv"]) * case["d"]
        turned = case["tokens"] * (case["hq"] + case["hkv"]) * case["part"]
        return {"bytes": 4 * n + 8 * case["tokens"], "flops": 3 * turned}
    old, new = _lengths(case)
    hkv, d, page = case["hkv"], case["d"], case["page"]
    row = hkv * d
    if case["op"] == "append":
        t, part = sum(new), sum(o % page for o in old)
        tokens = 4 * t * case["hq"] * d + 4 * t * row                       # q in and out, k and v in
        cached = 2 * t * row + 2 * part * row                              # new values out, the page's older ones in
        return {"bytes": tokens + cached + 4 * len(old) * _shown(case) * row, "flops": t * (3 * (case["hq"] + hkv) + 4 * hkv) * d}
    if case["op"] == "attend":
        window = case["window"] or 1 << 60
        seen = sum(min(o + n, n + window - 1) for o, n in zip(old, new))    # keys that some query of the step sees
        pairs = sum(sum(min(o + 1 + j, window) for j in range(n)) for o, n in zip(old, new))
        b = 2 * seen * row + 4 * sum(new) * case["hq"] * d + 4 * sum(new) * case["hq"] + 8 * hkv * seen // page
        return {"bytes": b + (8 * seen * hkv if case["weights"] else 0), "flops": 4 * pairs * case["hq"] * d}
    kept = sum(min(o, case["budget"]) for o in old)
    return {"bytes": 4 * sum(old) * hkv + 4 * kept * row + 8 * kept * hkv + 4 * len(old) * case["budget"] * row,
            "flops": 4 * kept * row}


def _shown(case):
    """Tokens of a sequence that are read back after an append: the pages that it touched, from the first of them on."""
    old, new = _lengths(case)
    return max(o + n - o // case["page"] * case["page"] for o, n in zip(old, new))


# ---- inputs -------------------------------------------------------------------------------------------------------

def frequencies(part, scaling):
    """(radians per position of each pair, factor on cos and sin) of the ways to scale for long contexts, in 64 bits."""
    f = [BASE ** (-2.0 * i / part) for i in range(part // 2)]
    if scaling == "linear":
        return [x / 4.0 for x in f], 1.0
    if scaling == "ntk":
        base = BASE * 4.0 ** (part / (part - 2.0))
        return [base ** (-2.0 * i / part) for i in range(part // 2)], 1.0
    if scaling == "yarn":       # fast pairs as they are, slow ones interpolated, a ramp between
        def pair(turns):
            return part * math.log(4096.0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(BASE))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), part - 1)
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(part // 2)]
        return [x / 32.0 * r + x * (1.0 - r) for x, r in zip(f, ramp)], 0.1 * math.log(32.0) + 1.0
    if scaling == "llama3":
        def one(x):
            wave = 2.0 * math.pi / x
            smooth = (8192.0 / wave - 1.0) / (4.0 - 1.0)
            return x / 8.0 if wave > 8192.0 / 1.0 else x if wave < 8192.0 / 4.0 else (1.0 - smooth) * x / 8.0 + smooth * x
        return [one(x) for x in f], 1.0
    return f, 1.0


SCALING = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "ntk": {"type": "ntk", "factor": 4.0},
    "yarn": {"type": "yarn", "factor": 32.0, "original_max_position": 4096},
    "llama3": {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position": 8192},
}


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _quantised(x, kind):
    """x [..., page, d] in 8 bits with a scale for each [...]."""
    scale = x.abs().amax(dim=(-1, -2)) / TOP[kind]
    y = (x / scale[..., None, None]).clamp(-TOP[kind], TOP[kind])
    return (y.round() if kind == "int8" else y).to(CACHE_TYPE[kind]), scale


def _cache(gen, pages, hkv, page, d, kind):
    k8 = torch.empty((pages, hkv, page, d), dtype=CACHE_TYPE[kind], device="cuda")
    v8, ks = torch.empty_like(k8), torch.empty((pages, hkv), device="cuda")
    vs = torch.empty_like(ks)
    loud = torch.ones(d, device="cuda")
    loud[:: d // 4] = 4.0
    step = max(1, 2 ** 26 // (hkv * page * d))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        k8[a:b], ks[a:b] = _quantised(_normal(gen, b - a, hkv, page, d) * loud, kind)
        v8[a:b], vs[a:b] = _quantised(_normal(gen, b - a, hkv, page, d), kind)
    return k8, v8, ks, vs


def _table(gen, need, spare=0):
    """A page table of scattered pages for sequences that need so many each."""
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen, device="cuda")
    table = torch.zeros((len(need), max(1, max(need))), dtype=torch.int64)
    at = 0
    host = order.tolist()
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(host[at:at + n], dtype=torch.int64)
        at += n
    return table.to("cuda"), order[at:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    io = IO_TYPE[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rotary":
        t, d = case["tokens"], case["d"]
        first = torch.randint(0, max(1, case["far"] - t), (1,), generator=gen, device="cuda")
        s["positions"] = first + torch.arange(t, device="cuda")
        s["q"], s["k"] = _normal(gen, t, case["hq"], d, dtype=io), _normal(gen, t, case["hkv"], d, dtype=io)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        freq, factor = frequencies(case["part"], case["scaling"])
        s["freq"], s["factor"] = torch.tensor(freq, dtype=torch.float64, device="cuda"), factor
        if own:
            import slora_b200 as sl
            s["table"] = sl.RotaryTable(d, case["part"], BASE, case["layout"], SCALING[case["scaling"]])
        return s
    hkv, d, page, kind = case["hkv"], case["d"], case["page"], case["kind"]
    old, new = _lengths(case)
    total = [o + n for o, n in zip(old, new)]
    kept = [min(o, case["budget"]) for o in old] if case["op"] == "evict" else []
    more = [-(-n // page) for n in kept]
    table, rest = _table(gen, [-(-n // page) for n in total], sum(more))
    s["page_table"] = table
    s["kv_len"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    s["q_len"] = torch.tensor(new, dtype=torch.int32, device="cuda")
    s["q_start"] = (torch.cumsum(s["q_len"], 0) - s["q_len"]).to(torch.int32)
    s["max_q"], s["max_kv"] = max(new), max(total)
    s["k8"], s["v8"], s["k_scale"], s["v_scale"] = _cache(gen, sum(-(-n // page) for n in total) + sum(more), hkv, page, d, kind)
    s["weights"] = None
    if case["op"] == "append":
        t = sum(new)
        s["q"], s["k"], s["v"] = (_normal(gen, t, h, d, dtype=io) for h in (case["hq"], hkv, hkv))
        s["q_out"] = torch.empty_like(s["q"])
        s["positions"] = torch.cat([torch.arange(o, o + n) for o, n in zip(old, new)]).to("cuda")
        freq, _ = frequencies(d, "none")
        s["freq"], s["factor"] = torch.tensor(freq, dtype=torch.float64, device="cuda"), 1.0
        s["shown_from"] = (torch.tensor(old, dtype=torch.int32) // page * page).to(torch.int32).to("cuda")
        s["shown"] = _shown(case)
    elif case["op"] == "attend":
        s["q"] = _normal(gen, sum(new), case["hq"], d, dtype=io)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((sum(new), case["hq"]), device="cuda")
        if case["weights"]:
            s["weights"] = torch.rand((s["k8"].size(0), hkv, page), generator=gen, device="cuda")
    else:
        s["weights"] = torch.empty((s["k8"].size(0), hkv, page), device="cuda").exponential_(generator=gen)
        dest = torch.zeros((len(kept), max(1, max(more))), dtype=torch.int64)
        at, host = 0, rest.tolist()
        for i, n in enumerate(more):
            dest[i, :n] = torch.tensor(host[at:at + n], dtype=torch.int64)
            at += n
        s["dest_table"] = dest.to("cuda")
        s["kept_len"] = torch.tensor(kept, dtype=torch.int32, device="cuda")
    if own:
        import slora_b200 as sl
        s["cache"] = sl.KvCache8.from_buffers([s["k8"]], [s["v8"]], [s["k_scale"]], [s["v_scale"]],
                                              None if s["weights"] is None else [s["weights"]])
        s["batch"] = sl.KvBatch(s["page_table"], s["kv_len"], s["q_start"], s["q_len"], s["max_q"], s["max_kv"])
        if case["op"] == "append":
            s["table"] = sl.RotaryTable(d, d, BASE, case["layout"])
        if case["op"] == "evict":
            zero = torch.zeros_like(s["kept_len"])
            s["dest"] = sl.KvBatch(s["dest_table"], s["kept_len"], zero, zero, 0, case["budget"])
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[case["op"]](s, case)


def _run_own(s, case):
    import slora_b200 as sl
    if case["op"] == "rotary":
        return list(sl.rotary(s["table"], s["positions"], s["q"], s["k"], q_out=s["q_out"], k_out=s["k_out"]))
    cache = s["cache"]
    if case["op"] == "append":
        q = cache.append(0, s["batch"], s["k"], s["v"], q=s["q"], q_out=s["q_out"], rope=(s["table"], s["positions"]))
        k, v = cache.read(0, s["batch"], s["q"].dtype, s["shown"], first=s["shown_from"])
        return [q, k, v, s["k_scale"], s["v_scale"]]
    if case["op"] == "attend":
        cache.attend(0, s["batch"], s["q"], out=s["out"], lse=s["lse"], window=case["window"], add_weights=case["weights"])
        return [s["out"], s["lse"]] + ([s["weights"]] if case["weights"] else [])
    kept = cache.evict(0, s["batch"], case["budget"], case["recent"], dest=s["dest"])
    k, v = cache.read(0, s["dest"], IO_TYPE[case["dtype"]], case["budget"])
    return [kept, k, v, s["k_scale"], s["v_scale"], s["weights"]]


def _turn(x, positions, freq, factor, layout):
    """Rotary embedding of x [tokens, heads, d] in 32 bits, its angles in 64."""
    angle = positions.double()[:, None] * freq
    c, n = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
    x = x.float()
    half = freq.numel()
    if layout == "half":
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * c - b * n, a * n + b * c, rest], -1)
    a, b, rest = x[..., 0:2 * half:2], x[..., 1:2 * half:2], x[..., 2 * half:]
    return torch.cat([torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2), rest], -1)


def _plain_rotary(s, case):
    return [_turn(s[n], s["positions"], s["freq"], s["factor"], case["layout"]).to(s[n].dtype) for n in ("q", "k")]


def _read(k8, scale, table, length, first, count, dtype):
    """Tokens first .. first + count of each sequence as the values they stand for, zero behind its end."""
    page = k8.size(2)
    at = first[:, None] + torch.arange(count, device="cuda")
    there = at < length[:, None]
    at = at.clamp(max=table.size(1) * page - 1)
    pages = torch.gather(table, 1, (at // page).long())
    x = _take(k8, (pages, slice(None), at % page)).float() * scale[pages][..., None]
    return torch.where(there[..., None, None], x, 0).to(dtype)


def _take(x8, at):
    """x8[at], the bytes moved as bytes."""
    return x8.view(torch.uint8)[at].view(x8.dtype)


def _put(x8, at, y):
    x8.view(torch.uint8)[at] = y.view(torch.uint8)


def _to8(x, scale, kind):
    """x / scale in 8 bits, the quotient in 64: values of a page that is scaled anew are often next to a border."""
    x = x.double() / torch.where(scale > 0, scale, 1).double()[..., None, None]
    x = x.clamp(-TOP[kind], TOP[kind])
    if kind == "int8":
        return x.round().to(torch.int8)
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent.clamp(min=-5) - 4)   # three bits behind the leading one
    return (torch.round(x / step) * step).to(torch.float8_e4m3fn)


def _plain_append(s, case):
    page, kind, hkv, d = case["page"], case["kind"], case["hkv"], case["d"]
    q = _turn(s["q"], s["positions"], s["freq"], s["factor"], case["layout"]).to(s["q"].dtype)
    k = _turn(s["k"], s["positions"], s["freq"], s["factor"], case["layout"])
    table, total, old = s["page_table"], s["kv_len"].long(), (s["kv_len"] - s["q_len"]).long()
    n = -(-s["shown"] // page)                                   # pages that a sequence's new tokens touch, at most
    at = s["shown_from"].long()[:, None] + torch.arange(n * page, device="cuda")
    isold, isnew = at < old[:, None], (at >= old[:, None]) & (at < total[:, None])
    block = at[:, ::page] // page
    touched = isnew.view(-1, n, page).any(-1)
    pages = torch.gather(table, 1, block.clamp(max=table.size(1) - 1))
    row = (s["q_start"].long()[:, None] + at - old[:, None]).clamp(0, k.size(0) - 1)
    for_block = (isold.view(-1, n, page)[..., None, :, None], isnew.view(-1, n, page)[..., None, :, None])
    for x, x8, scale in ((k, s["k8"], s["k_scale"]), (s["v"].float(), s["v8"], s["v_scale"])):
        x = x[row].view(-1, n, page, hkv, d).transpose(2, 3)     # [seqs, n, hkv, page, d]
        was = _take(x8, pages).float()
        s_old = torch.where(for_block[0][:, :, 0, 0], scale[pages], 0)
        s_new = torch.maximum(s_old, (torch.where(for_block[1], x.abs(), 0).amax((-1, -2)).double() / TOP[kind]).float())
        x = torch.where(for_block[1], x.double(), was.double() * s_old[..., None, None])
        y = _to8(x, s_new, kind)
        stay = ((s_new == s_old)[..., None, None] & for_block[0]) | ~(for_block[0] | for_block[1])
        y = torch.where(stay, _take(x8, pages).view(torch.uint8), y.view(torch.uint8)).view(x8.dtype)
        _put(x8, pages[touched], _take(y, touched))
        scale[pages[touched]] = s_new[touched]
    first = s["shown_from"].long()
    return [q] + [_read(a, b, table, total, first, s["shown"], q.dtype) for a, b in ((s["k8"], s["k_scale"]), (s["v8"], s["v_scale"]))] + \
        [s["k_scale"], s["v_scale"]]


def _plain_attend(s, case):
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    group, seqs, top = hq // hkv, case["seqs"], s["max_q"]
    old, new = (s["kv_len"] - s["q_len"]).long(), s["q_len"].long()
    j = torch.arange(top, device="cuda")
    row = (s["q_start"].long()[:, None] + j).clamp(max=s["q"].size(0) - 1)
    real = j < new[:, None]
    q = s["q"].float()[row].view(seqs, top, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, group * top, d)
    table = s["page_table"]
    length = table.size(1) * page

    def dense(x8, scale):
        return (_take(x8, table).float() * scale[table][..., None, None]).transpose(1, 2).reshape(seqs, hkv, length, d)

    score = q @ dense(s["k8"], s["k_scale"]).transpose(-1, -2) * d ** -0.5
    key, last = torch.arange(length, device="cuda"), old[:, None] + j
    seen = (key <= last[..., None]) & real[..., None]
    if case["window"]:
        seen &= key > last[..., None] - case["window"]
    seen = seen[:, None, None].expand(seqs, 1, group, top, length).reshape(seqs, 1, group * top, length)
    score = score.masked_fill_(~seen, -math.inf)
    high = score.amax(-1, keepdim=True)
    high = torch.where(high > -math.inf, high, 0)
    p = score.sub_(high).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1))
    out = (p @ dense(s["v8"], s["v_scale"])).view(seqs, hkv, group, top, d).permute(0, 3, 1, 2, 4).reshape(seqs, top, hq, d)
    lse = (total.log() + high).view(seqs, hkv, group, top).permute(0, 3, 1, 2).reshape(seqs, top, hq)
    s["out"][row[real]] = out[real].to(s["out"].dtype)
    s["lse"][row[real]] = lse[real]
    if not case["weights"]:
        return [s["out"], s["lse"]]
    w = p.sum(2).view(seqs, hkv, -1, page).transpose(1, 2)
    used = torch.arange(table.size(1), device="cuda") * page < s["kv_len"][:, None]
    s["weights"][table[used]] += w[used]
    return [s["out"], s["lse"], s["weights"]]


def _plain_evict(s, case):
    page, kind, budget = case["page"], case["kind"], case["budget"]
    table, n, dest = s["page_table"], s["kv_len"].long(), s["dest_table"]
    seqs, hkv = table.size(0), case["hkv"]
    w = s["weights"][table].transpose(1, 2).reshape(seqs, hkv, -1)
    at = torch.arange(w.size(-1), device="cuda")
    rank = w.masked_fill((at >= n[:, None] - case["recent"])[:, None], math.inf).masked_fill((at >= n[:, None])[:, None], -math.inf)
    kept = rank.sort(stable=True, dim=-1, descending=True).indices[..., :budget]
    if kept.size(-1) < budget:
        kept = torch.cat([kept, kept.new_zeros(seqs, hkv, budget - kept.size(-1))], -1)
    j = torch.arange(budget, device="cuda")
    there = (j < n[:, None])[:, None].expand_as(kept)
    kept = torch.where(there, kept, 1 << 40).sort(-1).values
    from_page = torch.gather(table[:, None].expand(-1, hkv, -1), 2, torch.where(there, kept, 0) // page)
    slot, head = torch.where(there, kept, 0) % page, torch.arange(hkv, device="cuda")[:, None]
    blocks = -(-budget // page)

    def in_blocks(x, fill):
        return torch.nn.functional.pad(x, (0, blocks * page - budget), value=fill).view(seqs, hkv, blocks, page)

    here = in_blocks(there, False)
    same = (in_blocks(kept == j, True) | ~here).all(-1)           # nothing in the block moves: it stays as it is
    used = here[..., 0][:, 0]
    to = dest[used[:, :dest.size(1)]]
    for x8, scale in ((s["k8"], s["k_scale"]), (s["v8"], s["v_scale"])):
        x = _take(x8, (from_page, head, slot)).double() * scale[from_page, head][..., None]
        x = torch.nn.functional.pad(torch.where(there[..., None], x, 0), (0, 0, 0, blocks * page - budget)).view(seqs, hkv, blocks, page, -1)
        s_new = torch.where(same, scale[in_blocks(from_page, 0)[..., 0], head], (x.abs().amax((-1, -2)) / TOP[kind]).float())
        y = _to8(x, s_new, kind)
        now = here.transpose(1, 2)[used][..., None]
        _put(x8, to, torch.where(now, y.view(torch.uint8).transpose(1, 2)[used], x8.view(torch.uint8)[to]))
        scale[to] = s_new.transpose(1, 2)[used]
    moved = in_blocks(torch.where(there, s["weights"][from_page, head, slot], 0), 0.0)
    s["weights"][to] = torch.where(here.transpose(1, 2)[used], moved.transpose(1, 2)[used], s["weights"][to])
    zero = torch.zeros_like(n)
    return [torch.where(there, kept, -1).to(torch.int32)] + \
        [_read(a, b, dest, s["kept_len"].long(), zero, budget, IO_TYPE[case["dtype"]]) for a, b in ((s["k8"], s["k_scale"]), (s["v8"], s["v_scale"]))] + \
        [s["k_scale"], s["v_scale"], s["weights"]]


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------

def _rotate64(x, pos, freq, factor, interleaved):
    """Each pair as a complex number times e^(i angle)."""
    n = freq.numel()
    z = torch.polar(torch.full((pos.numel(), n), factor, dtype=torch.float64, device="cuda"),
                    torch.outer(pos.double(), freq))[:, None]
    x = x.double().clone()
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * z
    x[..., one], x[..., two] = y.real, y.imag
    return x


def _round64(x, kind):
    if kind == "int8":
        return torch.round(x).clamp(-127, 127)
    m = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(m.clamp(min=2.0 ** -6))) - 3.0)      # e4m3: 3 bits behind the leading one
    return torch.sign(x) * torch.round(m / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return [_rotate64(s[n], s["positions"], s["freq"], s["factor"], case["layout"] == "interleaved") for n in ("q", "k")]
    hkv, d, page, kind = case["hkv"], case["d"], case["page"], case["kind"]
    old, new = _lengths(case)
    table, top = s["page_table"].tolist(), TOP[kind]
    ks, vs = s["k_scale"].double(), s["v_scale"].double()

    def values(i, n):
        """Sequence i's first n keys and values, [hkv, n, d]."""
        p = torch.tensor(table[i][:-(-n // page)], dtype=torch.int64, device="cuda")
        return [(_take(x, p).double() * sc[p][..., None, None]).transpose(0, 1).reshape(hkv, -1, d)[:, :n]
                for x, sc in ((s["k8"], ks), (s["v8"], vs))]

    if case["op"] == "append":
        inter = case["layout"] == "interleaved"
        fresh = [_rotate64(s["k"], s["positions"], s["freq"], 1.0, inter), s["v"].double()]
        shown = [torch.zeros((len(old), s["shown"], hkv, d), dtype=torch.float64, device="cuda") for _ in range(2)]
        at = 0
        for i, (o, n) in enumerate(zip(old, new)):
            start = o // page * page
            for x, x8, scale, show in zip(fresh, (s["k8"], s["v8"]), (ks, vs), shown):
                for b in range(start // page, -(-(o + n) // page)):
                    lo, hi, p = max(o, b * page), min(o + n, (b + 1) * page), table[i][b]
                    y = x[at + lo - o: at + hi - o].transpose(0, 1)                # [hkv, new tokens of the page, d]
                    kept = x8[p][:, :max(0, o - b * page)].double()
                    was = scale[p].clone() if kept.size(1) else torch.zeros_like(scale[p])
                    now = torch.maximum(was, (y.abs().amax((-1, -2)) / top).float().double())     # scales are held in 32 bits
                    ratio = torch.where(now == was, 1.0, was / now)[:, None, None]
                    every = torch.cat([torch.where(ratio == 1.0, kept, _round64(kept * ratio, kind)),
                                       _round64(y / now[:, None, None], kind)], 1) * now[:, None, None]
                    scale[p] = now
                    show[i, b * page - start: b * page - start + every.size(1)] = every.transpose(0, 1)
            at += n
        return [_rotate64(s["q"], s["positions"], s["freq"], 1.0, inter)] + shown + [ks, vs]
    if case["op"] == "attend":
        hq, group = case["hq"], case["hq"] // hkv
        out, lse = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), torch.empty(s["lse"].shape, dtype=torch.float64, device="cuda")
        w = None if s["weights"] is None else s["weights"].double()
        at = 0
        for i, (o, n) in enumerate(zip(old, new)):
            k, v = values(i, o + n)
            for a in range(0, n, 256):
                b = min(n, a + 256)
                q = s["q"][at + a: at + b].double().view(b - a, hkv, group, d).permute(1, 2, 0, 3)
                score = torch.einsum("hgqd,hkd->hgqk", q, k) / math.sqrt(d)
                place = torch.arange(o + n, device="cuda")
                mine = o + torch.arange(a, b, device="cuda")[:, None]
                hidden = (place > mine) | ((place <= mine - case["window"]) if case["window"] else False)
                score = score.masked_fill(hidden, -math.inf)
                z = torch.logsumexp(score, -1)
                p = torch.exp(score - z[..., None])
                out[at + a: at + b] = torch.einsum("hgqk,hkd->qhgd", p, v).reshape(b - a, hq, d)
                lse[at + a: at + b] = z.permute(2, 0, 1).reshape(b - a, hq)
                if w is not None:
                    pages = torch.tensor(table[i][:-(-(o + n) // page)], dtype=torch.int64, device="cuda")
                    add = torch.nn.functional.pad(p.sum((1, 2)), (0, pages.numel() * page - o - n))
                    w[pages] += add.view(hkv, -1, page).transpose(0, 1)
            at += n
        return [out, lse] + ([] if w is None else [w])
    budget, recent = case["budget"], case["recent"]
    dest, w = s["dest_table"].tolist(), s["weights"].double()
    shown = [torch.zeros((len(old), budget, hkv, d), dtype=torch.float64, device="cuda") for _ in range(2)]
    for i, n in enumerate(old):
        both = values(i, n)
        p = torch.tensor(table[i][:-(-n // page)], dtype=torch.int64, device="cuda")
        mine = s["weights"][p].transpose(0, 1).reshape(hkv, -1)[:, :n]
        m = min(n, budget)
        if n > budget:
            best = torch.argsort(mine[:, :n - recent], dim=1, descending=True, stable=True)[:, :budget - recent]
            tail = torch.arange(n - recent, n, device="cuda").expand(hkv, -1)
            keep = torch.cat([best, tail], 1).sort(1).values
        else:
            keep = torch.arange(n, device="cuda").expand(hkv, -1)
        for b in range(-(-m // page)):
            at = keep[:, b * page: min(m, (b + 1) * page)]
            still = (at == torch.arange(b * page, b * page + at.size(1), device="cuda")).all(1)
            for x, scale, show in zip(both, (ks, vs), shown):
                y = torch.gather(x, 1, at[..., None].expand(-1, -1, d))
                now = torch.where(still, scale[table[i][b]], (y.abs().amax((-1, -2)) / top).float().double())
                show[i, b * page: b * page + at.size(1)] = (_round64(y / now[:, None, None], kind) * now[:, None, None]).transpose(0, 1)
                scale[dest[i][b]] = now
            w[dest[i][b], :, :at.size(1)] = torch.gather(mine, 1, at).double()
    return [None] + shown + [ks, vs, w]
