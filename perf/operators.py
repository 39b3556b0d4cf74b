"""What is measured of the operators around a cache that is held in 8 bits, and their plain forms.

``store``      the keys and values of a step's tokens into a paged cache of e4m3 codes with one scale, a power of two, for each page and head
``attention``  a step's queries over such a cache: rows that decode one token, rows that bring a portion of a prompt, and both in one step
``tables``     a step's tables (which row and place a token has, where it is stored, each row's pages) from the lengths of its requests

``own`` false: elementary torch operations in 32 bits.  ``own`` true: the calls that a program makes of ``arle_b200.ops``.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
E4M3_MOST = 448.0
LOW, HIGH = -100, 119          # exponents that a scale may have


def listed():
    return [
        # one user's chat: every layer of every decoded token stores one key and one value; launch latency is all there is
        dict(name="store, one token", op="store", rows=1, portions=0, new=1, ctx=1500, nkv=8, hd=128, page=16, dtype="bfloat16", lens=1),
        # a full decode step of a server: 64 requests append one token each, most of them into a page that is partly filled
        dict(name="store, 64 decoded tokens", op="store", rows=64, portions=0, new=1, ctx=2000, nkv=8, hd=128, page=16, dtype="bfloat16", lens=2),
        # the engine's largest prompt step, cut from several requests at odd places
        dict(name="store, prompts of 15,000 tokens", op="store", rows=6, portions=6, new=4000, ctx=2500, nkv=8, hd=128, page=16, dtype="bfloat16", lens=3),
        # the 32-bit path with small heads and long pages: a prompt beside decoded tokens
        dict(name="store, float32, pages of 64", op="store", rows=9, portions=1, new=1001, ctx=900, nkv=4, hd=64, page=64, dtype="float32", lens=4),
        # one user's chat with a small model: few keys, so the time is the latency of one launch
        dict(name="attention, one row", op="attention", rows=1, portions=0, new=1, ctx=1000, nq=16, nkv=8, hd=128, page=16, window=0, sink=False,
             dtype="bfloat16", lens=5),
        # a server's decode step: 64 requests of ragged lengths
        dict(name="attention, 64 rows", op="attention", rows=64, portions=0, new=1, ctx=4096, nq=32, nkv=8, hd=128, page=16, window=0, sink=False,
             dtype="bfloat16", lens=6),
        # few requests with long documents, what an 8-bit cache is for
        dict(name="attention, 8 long rows", op="attention", rows=8, portions=0, new=1, ctx=32768, nq=32, nkv=8, hd=128, page=16, window=0, sink=False,
             dtype="bfloat16", lens=7),
        # small heads, a sliding window and sinks
        dict(name="attention, window and sinks", op="attention", rows=48, portions=0, new=1, ctx=5000, nq=16, nkv=4, hd=64, page=64, window=1024,
             sink=True, dtype="bfloat16", lens=8),
        # a mixed step: a prompt's next portion beside requests that decode
        dict(name="attention, mixed step", op="attention", rows=16, portions=1, new=509, ctx=2100, nq=32, nkv=8, hd=128, page=16, window=0, sink=False,
             dtype="bfloat16", lens=9),
        # a long prompt's last portion
        dict(name="attention, portion of 4,096", op="attention", rows=1, portions=1, new=4096, ctx=16384, nq=32, nkv=8, hd=128, page=16, window=0,
             sink=False, dtype="bfloat16", lens=10),
        # a small decode step's tables
        dict(name="tables, 8 rows", op="tables", rows=8, portions=0, new=1, ctx=2000, page=16, slots=64, lens=11),
        # the largest step: long prompts beside a full house of decoding requests
        dict(name="tables, 256 rows", op="tables", rows=256, portions=12, new=1500, ctx=16000, page=16, slots=300, lens=12),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["store", "store", "attention", "attention", "attention", "tables"])
    page = rng.choice([8, 16, 16, 32, 64])
    lens = rng.randrange(1 << 30)
    if op == "tables":
        rows = _log(rng, 1, 256)
        return dict(op=op, rows=rows, portions=rng.randint(0, min(rows, 12)), new=_log(rng, 2, 1500), ctx=_log(rng, 4, 16000), page=page,
                    slots=rows + rng.randint(0, 40), lens=lens)
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    nkv, hd = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 128, 80])
    if op == "store":
        portions = rng.choice([0, 1, rng.randint(1, 6)])
        rows = max(portions, _log(rng, 1, 64))
        return dict(op=op, rows=rows, portions=portions, new=_log(rng, 2, 4000 // max(1, portions)), ctx=_log(rng, 2, 2500), nkv=nkv, hd=hd, page=page,
                    dtype=dtype, lens=lens)
    group = rng.choice([1, 2, 4, 8])
    window = rng.choice([0, 0, _log(rng, 16, 2048)])
    form = rng.choice(["decode", "decode", "portion", "mixed"])
    if dtype == "float32" or hd == 80:      # what the general kernel takes: shorter rows
        rows, ctx, new = _log(rng, 1, 16), _log(rng, 2, 1000), _log(rng, 2, 60)
    elif form == "decode":
        rows = _log(rng, 1, 64)
        ctx, new = _log(rng, 2, min(32768, 262144 // rows)), 1
    else:
        rows, ctx, new = _log(rng, 2, 12), _log(rng, 2, 3000), _log(rng, 2, 700)
    portions = 0 if form == "decode" else 1
    rows = 1 if form == "portion" else rows
    return dict(op=op, rows=rows, portions=portions, new=new, ctx=max(ctx, new if portions else 1), nq=nkv * group, nkv=nkv, hd=hd, page=page, window=window,
                sink=rng.random() < 0.25, dtype=dtype, lens=lens)


def lengths(case):
    """(tokens held before the step, tokens of the step) of each row: the first ``portions`` rows bring portions, the others one token."""
    rng = random.Random(case["lens"])
    starts, news = [], []
    for r in range(case["rows"]):
        new = (case["new"] if r == 0 else rng.randint(max(1, case["new"] // 4), case["new"])) if r < case["portions"] else 1
        if case["op"] == "attention":      # ctx: what the longest row holds after the step
            keys = case["ctx"] if r == 0 else rng.randint(max(new, case["ctx"] // 3), max(new, case["ctx"]))
            starts.append(keys - new)
        else:                              # ctx: what the longest row holds before it
            starts.append(case["ctx"] if r == 0 else rng.randint(0, case["ctx"]))
        news.append(new)
    order = list(range(case["rows"]))
    rng.shuffle(order)
    return [starts[r] for r in order], [news[r] for r in order]


def visible(case, starts, news):
    """(pairs of a query and a key that it sees, keys that some query of a row sees) over all rows."""
    pairs = keys = 0
    for s, n in zip(starts, news):
        w = case["window"] or s + n
        full = max(0, min(n, s + n - w))               # queries that see w keys, the others fewer
        few = n - full
        pairs += full * w + sum(range(s + 1, s + few + 1))
        keys += s + n - max(0, s + 1 - w)
    return pairs, keys


def work(case):
    starts, news = lengths(case)
    T, R, ps = sum(news), case["rows"], case["page"]
    pages = [-(-(s + n) // ps) for s, n in zip(starts, news)]
    if case["op"] == "tables":
        held = [-(-s // ps) for s in starts]
        gained = sum(p - h for p, h in zip(pages, held))
        return {"bytes": 4 * (3 * R + 2 * gained + sum(held) + 2 * R + 1 + 4 * T + R * max(pages)), "flops": 0}
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "store":
        touched = sum(p - s // ps for p, s in zip(pages, starts))
        return {"bytes": 2 * T * case["nkv"] * case["hd"] * (size + 1) + 4 * T + 2 * 2 * 4 * touched * case["nkv"], "flops": 0}
    pairs, keys = visible(case, starts, news)
    io = 2 * T * case["nq"] * case["hd"] * size
    return {"bytes": io + 2 * keys * case["nkv"] * case["hd"] + 2 * 4 * -(-keys // ps) * case["nkv"] + 4 * sum(pages), "flops": 4 * pairs * case["nq"] * case["hd"]}


# ------------------------------------------------------------------ inputs
def _values(g, shape, dtype=torch.float32):
    """Keys or values as a layer makes them, [tokens, heads, size]: a few channels are much larger than the others, and tokens differ in size."""
    x = torch.randn(shape, generator=g, device=DEV)
    loud = torch.exp(0.7 * torch.randn(shape[1:], generator=g, device=DEV))
    size = torch.exp(0.4 * torch.randn((shape[0], 1, 1), generator=g, device=DEV))
    return (x * loud * size).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cache(g, case, pages):
    """Codes and scales of a cache whose pages are all written."""
    nkv, hd, ps = case["nkv"], case["hd"], case["page"]
    x = _values(g, (pages * ps, nkv, hd)).view(pages, ps, nkv, hd).transpose(1, 2)
    scale = _scale_of(x.abs().amax(dim=(2, 3)))
    return (x / scale[:, :, None, None]).to(torch.float8_e4m3fn).contiguous(), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 17)
    starts, news = lengths(case)
    R, T, ps = case["rows"], sum(news), case["page"]
    rows = [r for r in range(R) for _ in range(news[r])]
    places = [starts[r] + i for r in range(R) for i in range(news[r])]
    indptr = [0]
    for n in news:
        indptr.append(indptr[-1] + n)
    held, pages = [-(-s // ps) for s in starts], [-(-(s + n) // ps) for s, n in zip(starts, news)]
    total = sum(pages) + 3
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    width = max(pages)
    if case["op"] == "tables":
        slots = torch.randperm(case["slots"], generator=g, device=DEV)[:R].to(torch.int32)
        table = torch.full((case["slots"], width + 5), -1, dtype=torch.int32, device=DEV)
        at = torch.arange(width + 5, device=DEV)[None, :]
        h = _i32(held).long()
        first = torch.cumsum(h, 0) - h
        mine = torch.where(at < h[:, None], order[(first[:, None] + at).clamp(max=total - 1)], -1)
        table[slots.long()] = mine.to(torch.int32)
        gained = order[sum(held): sum(pages)].contiguous()
        out = {n: torch.full((k,), -7, dtype=torch.int32, device=DEV)
               for n, k in (("q_indptr", R + 1), ("kv_lens", R), ("positions", T), ("row_of_token", T), ("slot_of_token", T), ("slot_mapping", T), ("status", 1))}
        out["block_table"] = torch.full((R, width), -7, dtype=torch.int32, device=DEV)
        return dict(case=case, slots=slots, starts=_i32(starts), q_lens=_i32(news), new_pages=gained, page_table=table, num_pages=total, out=out)
    table = torch.full((R, width), -1, dtype=torch.int32)
    cut, host = 0, order.cpu()
    for r in range(R):
        table[r, : pages[r]] = host[cut: cut + pages[r]]
        cut += pages[r]
    slot = table[torch.tensor(rows), torch.tensor(places) // ps] * ps + torch.tensor(places, dtype=torch.int32) % ps
    dtype = DTYPES[case["dtype"]]
    k_cache, k_scale = _cache(g, case, total)
    v_cache, v_scale = _cache(g, case, total)
    s = dict(case=case, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, q_indptr=_i32(indptr), kv_lens=_i32([a + b for a, b in zip(starts, news)]),
             positions=_i32(places), row_of_token=_i32(rows), block_table=table.to(DEV), slot_mapping=slot.to(torch.int32).to(DEV), q_lens=news, most=max(news))
    if case["op"] == "store":
        # the rows of a packed projection q | k | v, as the engine's product leaves them
        nkv, hd = case["nkv"], case["hd"]
        qkv = torch.empty((T, 4 * nkv * hd), dtype=dtype, device=DEV)
        qkv[:, 2 * nkv * hd:] = torch.cat([_values(g, (T, nkv, hd)).view(T, -1), _values(g, (T, nkv, hd)).view(T, -1)], dim=1).to(dtype)
        s.update(k=qkv[:, 2 * nkv * hd: 3 * nkv * hd], v=qkv[:, 3 * nkv * hd:])
    else:
        s["q"] = torch.randn((T, case["nq"] * case["hd"]), generator=g, device=DEV).to(dtype)
        s["out"] = torch.empty_like(s["q"])
        s["sinks"] = torch.randn(case["nq"], generator=g, device=DEV) if case["sink"] else None
    return s


# ------------------------------------------------------------------ plain forms
def _scale_of(most):
    """The smallest power of two s with most / s <= 448 = 1.75 * 2^8 (most = f * 2^e with f in [0.5, 1): 2^(e - 9), doubled where f > 0.875)."""
    f, e = torch.frexp(most)
    e = torch.where(most > 0, e - 9 + (f > 0.875).to(e.dtype), LOW).clamp(LOW, HIGH)
    return torch.ldexp(torch.ones_like(most), e)


def _codes(x, scale):
    return (x / scale).clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn)


def _store_plain(x, cache, scale, s):
    case = s["case"]
    nkv, hd, ps = case["nkv"], case["hd"], case["page"]
    pages = cache.shape[0]
    x = x.reshape(-1, nkv, hd).float()
    page, off = (s["slot_mapping"] // ps).long(), (s["slot_mapping"] % ps).long()
    most = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dim=2)
    of_page = torch.zeros((pages, nkv), device=x.device).scatter_reduce_(0, page[:, None].expand(-1, nkv), most, "amax")
    first = torch.full((pages,), ps, dtype=torch.long, device=x.device).scatter_reduce_(0, page, off, "amin")
    new = _scale_of(of_page)
    now = torch.where(first[:, None] == ps, scale, torch.where(first[:, None] == 0, new, torch.maximum(scale, new)))
    # the page that a row's first token goes to holds older tokens in front of it: their codes follow the page's scale
    lead = s["q_indptr"][:-1].long()
    old = page[lead]
    was = cache[old].float() * (scale[old] / now[old])[:, :, None, None]
    older = torch.arange(ps, device=x.device)[None, None, :, None] < off[lead][:, None, None, None]
    bits = cache.view(torch.uint8)
    bits[old] = torch.where(older, was.clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn).view(torch.uint8), bits[old])
    bits[page, :, off] = _codes(x, now[page][:, :, None]).view(torch.uint8)
    scale.copy_(now)


def _attention_plain(s):
    case = s["case"]
    nq, nkv, hd, ps, T = case["nq"], case["nkv"], case["hd"], case["page"], s["q"].shape[0]
    R, W = s["block_table"].shape
    n, g = s["most"], nq // nkv
    table = s["block_table"].clamp(min=0).long()

    def read(cache, scale):        # [R, nkv, W * ps, hd]
        return (cache[table].float() * scale[table][:, :, :, None, None]).transpose(1, 2).reshape(R, nkv, W * ps, hd)

    at = s["q_indptr"][:-1, None].long() + torch.arange(n, device=DEV)[None, :]
    mine = at < s["q_indptr"][1:, None].long()
    at = at.clamp(max=T - 1)
    q = s["q"][at].float().view(R, n, nkv, g, hd).permute(0, 2, 3, 1, 4).reshape(R, nkv, g * n, hd)
    scores = torch.matmul(q, read(s["k_cache"], s["k_scale"]).transpose(2, 3)).view(R, nkv, g, n, W * ps) * hd ** -0.5
    place = s["positions"][at][:, None, None, :, None]
    key = torch.arange(W * ps, device=DEV)
    seen = (key <= place) & mine[:, None, None, :, None]
    if case["window"]:
        seen &= key > place - case["window"]
    scores = scores.masked_fill(~seen, -math.inf)
    most = scores.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    sink = s["sinks"].view(1, nkv, g, 1, 1) if s["sinks"] is not None else None
    if sink is not None:
        most = torch.maximum(most, sink)
    p = torch.exp(scores - most)
    total = p.sum(dim=-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - most)
    p = (p / total.clamp(min=1e-30)).view(R, nkv, g * n, W * ps)
    o = torch.matmul(p, read(s["v_cache"], s["v_scale"])).view(R, nkv, g, n, hd).permute(0, 3, 1, 2, 4).reshape(R, n, nq * hd)
    row = s["row_of_token"].long()
    s["out"].copy_(o[row, torch.arange(T, device=DEV) - s["q_indptr"].long()[row]])


def _tables_plain(s):
    out, ps = s["out"], s["case"]["page"]
    T, W = out["positions"].shape[0], out["block_table"].shape[1]
    slots, starts, lens = s["slots"].long(), s["starts"].long(), s["q_lens"].long()
    ends = starts + lens
    until = torch.cumsum(lens, 0)
    held, pages = (starts + ps - 1) // ps, (ends + ps - 1) // ps
    gained = pages - held
    first = torch.cumsum(gained, 0) - gained
    table = s["page_table"]
    at = torch.arange(table.shape[1], device=DEV)[None, :]
    mine = table[slots].long()
    fresh = s["new_pages"].long()[(first[:, None] + at - held[:, None]).clamp(0, max(s["new_pages"].shape[0] - 1, 0))] if s["new_pages"].shape[0] else mine
    mine = torch.where((at >= held[:, None]) & (at < pages[:, None]), fresh, mine)
    table[slots] = mine.to(torch.int32)
    out["block_table"].copy_(torch.where(at < pages[:, None], mine, -1)[:, :W])
    row = torch.searchsorted(until, torch.arange(T, device=DEV), right=True)
    place = starts[row] + torch.arange(T, device=DEV) - (until - lens)[row]
    out["q_indptr"].copy_(torch.cat([torch.zeros_like(until[:1]), until]))
    out["kv_lens"].copy_(ends)
    out["positions"].copy_(place)
    out["row_of_token"].copy_(row)
    out["slot_of_token"].copy_(slots[row])
    out["slot_mapping"].copy_(mine[row, place // ps] * ps + place % ps)
    out["status"].zero_()


# ------------------------------------------------------------------ the framework's calls
def _batch(s):
    """What the attention is told of a step: an engine's step context has these names.  Made once a step, for all its layers."""
    from types import SimpleNamespace

    from arle_b200.engine.batch import Workspace

    lens = [int(n) for n in s["kv_lens"].cpu()]
    return SimpleNamespace(q_indptr=s["q_indptr"], kv_lens=s["kv_lens"], q_lens=s["q_lens"], kv_lens_host=lens, num_rows=len(lens), max_q_len=s["most"],
                           max_kv_len=max(lens), num_single=sum(n == 1 for n in s["q_lens"]), ws=Workspace(DEV), memo={})


def run(state):
    s, case = state, state["case"]
    if own:
        from arle_b200 import ops
    if case["op"] == "store":
        if own:
            ops.store_q8(s["k"], s["v"], s["slot_mapping"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], case["nkv"], case["hd"], case["page"])
        else:
            _store_plain(s["k"], s["k_cache"], s["k_scale"], s)
            _store_plain(s["v"], s["v_cache"], s["v_scale"], s)
        return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    if case["op"] == "tables":
        if own:
            o = s["out"]
            ops.step_tables(s["slots"], s["starts"], s["q_lens"], s["new_pages"], s["page_table"], s["num_pages"], case["page"], o["q_indptr"], o["kv_lens"],
                            o["positions"], o["row_of_token"], o["slot_of_token"], o["slot_mapping"], o["block_table"], o["status"])
        else:
            _tables_plain(s)
        return {**s["out"], "page_table": s["page_table"]}
    if own:
        if "batch" not in s:
            s["batch"] = _batch(s)
        ops.paged_attention_q8(s["q"], s["out"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["positions"], s["row_of_token"], s["block_table"],
                               case["nq"], case["nkv"], case["hd"], case["page"], case["hd"] ** -0.5, case["window"] or None, batch=s["batch"], sink=s["sinks"])
    else:
        _attention_plain(s)
    return s["out"]


# ------------------------------------------------------------------ in 64 bits
def _exact_store(x, cache, scale, s):
    case = s["case"]
    ps, nkv, hd = case["page"], case["nkv"], case["hd"]
    values = cache.double() * scale.double()[:, :, None, None]
    x = x.double().reshape(-1, nkv, hd)
    slots, cuts = s["slot_mapping"].tolist(), s["q_indptr"].tolist()
    scale, codes = scale.double().clone(), cache.double().clone()
    parts = []                                     # (page, first place, first token, tokens)
    for a, b in zip(cuts[:-1], cuts[1:]):
        while a < b:
            off = slots[a] % ps
            n = min(ps - off, b - a)
            parts.append((slots[a] // ps, off, a, n))
            a += n
    page, off, tok, num = (torch.tensor(c, device=DEV) for c in zip(*parts))
    i = torch.arange(ps, device=DEV)[None, :]
    new = (i >= off[:, None]) & (i < (off + num)[:, None])                      # [parts, ps]
    rows = x[(tok[:, None] + i - off[:, None]).clamp(0, x.shape[0] - 1)].transpose(1, 2)      # [parts, nkv, ps, hd]
    most = torch.where(new[:, None, :, None], rows.abs(), 0.0).amax(dim=(2, 3))
    want = torch.full_like(most, 2.0 ** LOW)
    least = torch.ceil(torch.log2((most / E4M3_MOST).clamp(min=2.0 ** -140)))
    for step in (0.0, 1.0):                        # a logarithm may be off in its last place: the least power that holds the largest value
        cand = torch.exp2((least - 1 + step).clamp(LOW, HIGH))
        want = torch.where((most / cand <= E4M3_MOST) & (want * E4M3_MOST < most), cand, want)
    want = torch.where(want * E4M3_MOST < most, torch.exp2((least + 1).clamp(LOW, HIGH)), want)
    now = torch.where(off[:, None] == 0, want, torch.maximum(scale[page], want))
    merged = torch.where(new[:, None, :, None], rows, values[page])
    fresh = (merged / now[:, :, None, None]).clamp(-E4M3_MOST, E4M3_MOST).float().to(torch.float8_e4m3fn).double()
    kept = new | (i < off[:, None])
    codes[page] = torch.where(kept[:, None, :, None], fresh, codes[page])
    scale[page] = now
    return codes, scale


def _exact_attention(s):
    case = s["case"]
    nq, nkv, hd, ps = case["nq"], case["nkv"], case["hd"], case["page"]
    g = nq // nkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    cuts, lens = s["q_indptr"].tolist(), s["kv_lens"].tolist()
    for r, length in enumerate(lens):
        a, b = cuts[r], cuts[r + 1]
        pages = s["block_table"][r, : -(-length // ps)].long()
        j = torch.arange(length, device=DEV)
        p = torch.arange(length - (b - a), length, device=DEV)
        hide = j[None, :] > p[:, None]
        if case["window"]:
            hide |= j[None, :] <= p[:, None] - case["window"]
        for h in range(nkv):
            k = (s["k_cache"][pages, h].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, hd)[:length]
            v = (s["v_cache"][pages, h].double() * s["v_scale"][pages, h].double()[:, None, None]).reshape(-1, hd)[:length]
            for i in range(h * g, h * g + g):
                z = s["q"][a:b, i * hd: i * hd + hd].double() @ k.T / math.sqrt(hd)
                z[hide] = -math.inf
                if s["sinks"] is not None:
                    z = torch.cat([z, s["sinks"][i].double().expand(b - a, 1)], dim=1)
                w = torch.softmax(z, dim=1)[:, :length]
                out[a:b, i * hd: i * hd + hd] = w @ v
    return out


def exact(case, seed):
    if case["op"] == "tables":
        return None                                # whole numbers
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    (k, ks), (v, vs) = _exact_store(s["k"], s["k_cache"], s["k_scale"], s), _exact_store(s["v"], s["v_cache"], s["v_scale"], s)
    return {"k_cache": k, "v_cache": v, "k_scale": ks, "v_scale": vs}
