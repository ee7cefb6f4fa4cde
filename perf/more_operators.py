"""The operators of a paged KV cache in 8 and 4 bits, and of sequences that
share their first pages, as measurable cases.

A quantised pool holds codes (``fp8``: e4m3, ``int8``, or ``fp4``: e2m1, two to
a byte, the lower half first) and, for every 32 of a row's dims, a power of two:
a byte e, 2^(e - 127), 255 for a block that holds an infinity or a NaN.  A
block's power is the smallest that keeps its largest magnitude within the
format (448, 127, 6), 2^-117 at least.

Four kinds of case, all through the public entry points of ``ops``:

- ``attention``: a batch of new tokens attends its sequences' rows in such pools
  (``ops.paged_attention``);
- ``store``: the norm and the rotation of queries and keys, with keys and values
  quantised as they are written (``ops.qk_norm_rope``), and the written rows
  read back (``ops.read_pages``);
- ``read``: whole sequences read back into contiguous 16-bit rows, as the index
  build takes them (``ops.read_pages``);
- ``shared``: a step of sequences that were forked from a few prompts: the pages
  that they share are found (``ops.share_prefixes``) and attended once for all
  of them, in each layer (``ops.paged_attention``).

``run`` is the plain form (elementary torch operations, 32-bit arithmetic)
unless ``own`` is set.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
THETA = 500000.0
BLOCK = 32
LARGEST = {"fp8": 448.0, "int8": 127.0, "fp4": 6.0}
FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # One new token of one 128k sequence: streaming K and V in 8 bits.
        _attention("q_decode_128k", [131072], [1]),
        # A decode batch of sequences at very different lengths, eight query
        # heads per KV head, rows of a token together, whole numbers as codes.
        _attention("q_decode_batch", _spread(40, 300, 40000), [1] * 40, kv_heads=4, groups=8, layout="tokens",
                   fmt="int8"),
        # The smallest call: a short sequence's next token; launches count.
        _attention("q_decode_small", [519], [1], page=8),
        # Long sequences in 4 bits, three drafted tokens each verified, half
        # precision, 64-wide heads.
        _attention("q_verify_fp4", _spread(12, 4000, 60000), [3] * 12, dim=64, page=32, dtype="fp16", fmt="fp4"),
        # Chunked prefill: the last 4096 tokens of a 16k prompt.
        _attention("q_chunk_16k", [16384], [4096]),
        # One token of each of 24 sequences normed, rotated, stored, read.
        _store("q_store_decode", _spread(24, 200, 100000), [1] * 24, fmt="int8"),
        # A prefill chunk's, ragged, with rows behind the last sequence.
        _store("q_store_chunk", [32768, 1000, 5003], [8192, 1000, 1337], pad=23),
        # A 32k sequence handed over to the retrieval index.
        _read("q_read_32k", [32768]),
        # Four short sequences of 64-wide heads in 4 bits.
        _read("q_read_small", [130, 7, 300, 65], dim=64, fmt="fp4", kv_heads=2, page=8, dtype="fp16"),
        # 64 requests behind one system prompt of 8k tokens.
        _shared("shared_prompt", [8192], 64, 20, 600),
        # Beam search: four prompts of eight beams in a quantised cache.
        _shared("shared_beams", [20001, 777, 4096, 12003], 8, 1, 300, fmt="fp8", kv_heads=4, groups=8, layers=1),
        # Two samples of one short prompt.
        _shared("shared_pair", [1500], 2, 10, 90, page=8, layers=1),
    ]


def _attention(name, lens, news, kv_heads=8, groups=4, dim=128, page=16, layout="heads", window=0, sinks=0,
               dtype="bf16", fmt="fp8", pad=0):
    return dict(name=name, kind="attention", lens=_text(lens), news=_text(news), kv_heads=kv_heads, groups=groups,
                dim=dim, page=page, layout=layout, window=window, sinks=sinks, dtype=dtype, fmt=fmt, pad=pad)


def _store(name, lens, news, kv_heads=8, groups=4, dim=128, page=16, layout="heads", dtype="bf16", fmt="fp8",
           rotary=None, interleaved=False, pad=0, norm=True):
    return dict(name=name, kind="store", lens=_text(lens), news=_text(news), kv_heads=kv_heads, groups=groups, dim=dim,
                page=page, layout=layout, dtype=dtype, fmt=fmt, rotary=dim if rotary is None else rotary,
                interleaved=interleaved, pad=pad, norm=norm)


def _read(name, lens, kv_heads=8, dim=128, page=16, layout="heads", dtype="bf16", fmt="fp8"):
    return dict(name=name, kind="read", lens=_text(lens), kv_heads=kv_heads, dim=dim, page=page, layout=layout,
                dtype=dtype, fmt=fmt)


def _shared(name, prompts, width, lo, hi, new=1, kv_heads=8, groups=4, dim=128, page=16, layout="heads", dtype="bf16",
            fmt="", layers=2):
    """Each prompt forked into ``width`` sequences, which have ``lo`` to ``hi`` rows of their own."""
    own_rows = [max(v, new) for v in _spread(len(prompts) * width, lo, hi)]
    return dict(name=name, kind="shared", prompts=_text(prompts), width=width, own=_text(own_rows), new=new,
                kv_heads=kv_heads, groups=groups, dim=dim, page=page, layout=layout, dtype=dtype, fmt=fmt,
                layers=layers)


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")] if text else []


def _spread(n, lo, hi):
    """n lengths spread evenly over the logarithm of lo..hi, odd ones among
    them, in an order that mixes long and short."""
    vals = [int(round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / max(n - 1, 1)))) for i in range(n)]
    return [vals[(i * 7) % n] if math.gcd(7, n) == 1 else vals[i] for i in range(n)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention"] * 4 + ["shared"] * 3 + ["store"] * 2 + ["read"])
    dim = rng.choice([64, 128, 128])
    layout = rng.choice(["heads", "tokens"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    fmt = rng.choice(["fp8", "fp8", "int8", "fp4"])
    if kind == "read":
        lens = [_log(rng, 1, 30000) for _ in range(rng.choice([1, 1, 2, 5, 9]))]
        lens = [min(v, 120000 // len(lens)) for v in lens]
        return _strip(_read("", lens, rng.choice([1, 2, 4, 8]), dim, rng.choice([8, 16, 64]), layout, dtype, fmt))
    if kind == "store":
        if rng.random() < 0.4:
            lens = [_log(rng, 1, 100000) for _ in range(rng.randint(1, 64))]
            news = [1] * len(lens)
        else:
            lens = [_log(rng, 100, 20000) for _ in range(rng.choice([1, 3, 17]))]
            news = [_log(rng, 1, max(1, min(v, 8000 // len(lens)))) for v in lens]
        # 4 bits: keys that were normed and rotated before
        plain = fmt == "fp4"
        rotary = 0 if plain else rng.choice([dim, dim, dim // 2])
        return _strip(_store("", lens, news, rng.choice([1, 2, 4, 8]), rng.choice([1, 4, 5, 8]), dim,
                             rng.choice([8, 16, 64]), layout, dtype, fmt, rotary, rng.random() < 0.3,
                             rng.choice([0, 0, 9]), not plain and rng.random() < 0.8))
    groups = rng.choice([1, 2, 4, 5, 7, 8, 16])
    kv_heads = rng.choice([1, 2, 4, 8])
    page = rng.choice([8, 16, 16, 32, 128])
    if kind == "shared":
        prompts = [_log(rng, 10, 20000) for _ in range(rng.choice([1, 1, 2, 4]))]
        width = rng.randint(2, 64 // len(prompts))
        lo = _log(rng, 1, 200)
        hi = _log(rng, lo + 1, 1500)
        return _strip(_shared("", prompts, width, lo, hi, rng.choice([1, 1, 1, 3, 5]), kv_heads, groups, dim, page,
                              layout, dtype, rng.choice(["", "", fmt]), rng.choice([1, 2])))
    window, sinks = rng.choice([(0, 0), (0, 0), (128, 4), (1000, 0), (4096, 32)])
    form = rng.choice(["decode", "batch", "few", "chunk", "mixed"])
    if form == "decode":
        lens = [_log(rng, 1, 131072)]
        news = [1]
    elif form == "batch":
        lens = [_log(rng, 1, 30000) for _ in range(rng.randint(2, 48))]
        news = [1] * len(lens)
    elif form == "few":
        lens = [_log(rng, 50, 20000) for _ in range(rng.randint(1, 24))]
        news = [min(v, rng.randint(2, 9)) for v in lens]
    elif form == "chunk":
        lens = [_log(rng, 100, 16000)]
        news = [_log(rng, 16, min(lens[0], 2048))]
    else:
        lens = [_log(rng, 1, 12000) for _ in range(rng.randint(3, 12))]
        news = [rng.choice([1, 1, 1, _log(rng, 1, min(v, 300))]) for v in lens]
    return _strip(_attention("", lens, news, kv_heads, groups, dim, page, layout, window, sinks, dtype, fmt,
                             rng.choice([0, 0, 7])))


def _strip(case):
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------ blocks --

def _encode(x, fmt):
    """Codes and exponents of values [..., dim] in 32 bits."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1)
    frac, e = torch.frexp(top)   # top = frac 2^e, frac in [0.5, 1)
    lead, e_top = math.frexp(LARGEST[fmt])
    k = (e - e_top + (frac > lead)).clamp(min=-117)
    k = torch.where(top > 0, k, -117)
    y = blocks * ((127 - k) << 23).view(torch.float32)[..., None]   # 2^-k, exactly
    if fmt == "fp8":
        codes = y.to(torch.float8_e4m3fn).flatten(-2)
    elif fmt == "int8":
        codes = y.round().to(torch.int8).flatten(-2)
    else:   # to the nearest of FP4, ties to the even code
        a = y.abs()
        c = torch.zeros_like(a, dtype=torch.uint8)
        for i, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
            c += (a >= mid) if i % 2 else (a > mid)
        c = (c + 8 * torch.signbit(y).to(torch.uint8)).flatten(-2)
        codes = c[..., 0::2] + 16 * c[..., 1::2]
    bad = ~torch.isfinite(top)
    e = torch.where(bad, 255, k + 127).to(torch.uint8)
    return codes, e


def _decode(codes, exponents, fmt):
    """The values in 32 bits."""
    if fmt == "fp4":
        table = torch.tensor(FP4 + [-v for v in FP4], device=codes.device)
        x = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)
    else:
        x = codes.float()
    scale = (exponents.int() << 23).view(torch.float32)
    scale = torch.where(exponents == 255, math.nan, scale)
    return (x.unflatten(-1, (-1, BLOCK)) * scale[..., None]).flatten(-2)


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _table(lens, page, gen, slack=1.2):
    """Random distinct pages of a pool for each sequence: (table int32 with -1
    past a sequence's pages, pages in the pool)."""
    held = [-(-n // page) for n in lens]
    pool = max(int(sum(held) * slack), sum(held) + 2, 4)
    ids = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(max(held), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, pool


def _starts(news):
    out = [0]
    for n in news:
        out.append(out[-1] + n)
    return out


def _order(t, layout):
    """[pages, heads, page, ...], the rows of a token together in memory where
    the layout says so."""
    return t if layout == "heads" else t.transpose(1, 2).contiguous().transpose(1, 2)


def _pool(case, pages, gen, spread):
    """A pool of keys or values, codes and exponents in a quantised one; spread:
    the log-normal factor of each head's channels."""
    H, page, D, fmt = case["kv_heads"], case["page"], case["dim"], case["fmt"]
    factor = torch.exp(spread * torch.randn((H, 1, D), generator=gen, device=DEV))
    step = max(1, (1 << 26) // (H * page * D))
    parts = []
    for p in range(0, pages, step):
        x = torch.randn((min(step, pages - p), H, page, D), generator=gen, device=DEV) * factor
        parts.append(_encode(x, fmt) if fmt else (x.to(DTYPES[case["dtype"]]),))
    return tuple(_order(torch.cat(t), case["layout"]) for t in zip(*parts))


def _empty_pool(case, pages):
    H, page, D, fmt = case["kv_heads"], case["page"], case["dim"], case["fmt"]
    code = {"fp8": torch.float8_e4m3fn, "int8": torch.int8, "fp4": torch.uint8}[fmt]
    codes = torch.zeros((pages, H, page, D // 2 if fmt == "fp4" else D), dtype=code, device=DEV)
    exps = torch.full((pages, H, page, D // BLOCK), 127, dtype=torch.uint8, device=DEV)
    return _order(codes, case["layout"]), _order(exps, case["layout"])


def prepare(case, seed):
    return {"attention": _prepare_attention, "store": _prepare_store, "read": _prepare_read,
            "shared": _prepare_shared}[case["kind"]](case, seed)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _queries(case, n, gen):
    return torch.randn((n, case["kv_heads"] * case["groups"], case["dim"]), generator=gen,
                       device=DEV).to(DTYPES[case["dtype"]])


def _results(case, n):
    heads = case["kv_heads"] * case["groups"]
    return (torch.zeros((n, heads, case["dim"]), dtype=DTYPES[case["dtype"]], device=DEV),
            torch.zeros((n, heads), dtype=torch.float32, device=DEV))


def _prepare_attention(case, seed):
    gen = _gen(seed)
    lens, news = _ints(case["lens"]), _ints(case["news"])
    start = _starts(news)
    n = start[-1] + case["pad"]
    state = dict(case=case, lens_host=lens, start_host=start, q=_queries(case, n, gen))
    state["table"], pool = _table(lens, case["page"], gen)
    state["k"], state["v"] = _pool(case, pool, gen, 0.5), _pool(case, pool, gen, 0.0)
    state["lens"], state["start"] = _i32(lens), _i32(start)
    state["out"], state["lse"] = _results(case, n)
    return state


def _prepare_store(case, seed):
    gen = _gen(seed)
    lens, news = _ints(case["lens"]), _ints(case["news"])
    H, G, D, page, dt = case["kv_heads"], case["groups"], case["dim"], case["page"], DTYPES[case["dtype"]]
    start = _starts(news)
    n = start[-1] + case["pad"]
    state = dict(case=case, lens_host=lens, start_host=start)
    # one projection's output: queries, keys and values of a token in one row
    qkv = (2.0 * torch.randn((n, (H * G + 2 * H) * D), generator=gen, device=DEV)).to(dt)
    state["q"] = qkv[:, :H * G * D].view(n, H * G, D)
    state["k"] = qkv[:, H * G * D:(H * G + H) * D].view(n, H, D)
    state["v"] = qkv[:, (H * G + H) * D:].view(n, H, D)
    weight = lambda: (1.0 + 0.2 * torch.randn((D,), generator=gen, device=DEV)).to(dt) if case["norm"] else None
    state["qw"], state["kw"] = weight(), weight()
    r = case["rotary"]
    freq = THETA ** (-torch.arange(0, r // 2, dtype=torch.float64, device=DEV) * 2.0 / max(r, 1))
    state["inv_freq"] = freq.float() if r else None
    state["q_out"] = torch.zeros((n, H * G, D), dtype=dt, device=DEV)
    state["table"], pool = _table(lens, page, gen)
    state["key_pages"], state["value_pages"] = _empty_pool(case, pool), _empty_pool(case, pool)
    pos = [lens[s] - news[s] + i for s in range(len(news)) for i in range(news[s])]
    seq = torch.tensor([s for s in range(len(news)) for _ in range(news[s])], device=DEV)
    state["positions"] = torch.tensor(pos, device=DEV)
    state["slots"] = (state["table"][seq, state["positions"] // page].long(), state["positions"] % page)
    state["rows"] = max(news)
    state["lens"], state["start"] = _i32(lens), _i32(start)
    state["first"] = _i32([a - b for a, b in zip(lens, news)])
    return state


def _prepare_read(case, seed):
    gen = _gen(seed)
    lens = _ints(case["lens"])
    state = dict(case=case, lens_host=lens, start_host=[0] * (len(lens) + 1))
    state["table"], pool = _table(lens, case["page"], gen)
    state["k"], state["v"] = _pool(case, pool, gen, 0.5), _pool(case, pool, gen, 0.0)
    state["lens"], state["start"] = _i32(lens), _i32(state["start_host"])
    shape = (len(lens), case["kv_heads"], max(lens), case["dim"])
    state["keys"] = torch.zeros(shape, dtype=DTYPES[case["dtype"]], device=DEV)
    state["values"] = torch.zeros_like(state["keys"])
    return state


def _prepare_shared(case, seed):
    gen = _gen(seed)
    prompts, width, own_rows, page = _ints(case["prompts"]), case["width"], _ints(case["own"]), case["page"]
    lens = [prompts[i // width] + n for i, n in enumerate(own_rows)]
    held = [-(-n // page) for n in lens]
    pool = int(1.1 * sum(held)) + 4
    ids = torch.randperm(pool, generator=gen, device=DEV).cpu().tolist()
    table = torch.full((len(lens), max(held)), -1, dtype=torch.int32)
    take = iter(ids)
    for s, n in enumerate(held):   # a prompt's full pages are held by all of its sequences
        same = prompts[s // width] // page if s % width else 0
        if same:
            table[s, :same] = table[s - s % width, :same]
        table[s, same:n] = torch.tensor([next(take) for _ in range(n - same)], dtype=torch.int32)
    used = pool - len(list(take))
    rank = torch.full((pool,), -1, dtype=torch.int32)   # no pages that nobody holds but a few
    rank[torch.tensor(sorted(ids[:used]), dtype=torch.long)] = torch.arange(used, dtype=torch.int32)
    table = torch.where(table >= 0, rank[table.clamp(min=0).long()], -1)
    start = _starts([case["new"]] * len(lens))
    state = dict(case=case, lens_host=lens, start_host=start, table=table.to(DEV), lens=_i32(lens), start=_i32(start))
    state["layers"] = []
    for _ in range(case["layers"]):
        out, lse = _results(case, start[-1])
        state["layers"].append(dict(q=_queries(case, start[-1], gen), k=_pool(case, used + 2, gen, 0.5),
                                    v=_pool(case, used + 2, gen, 0.0), out=out, lse=lse))
    return state


# --------------------------------------------------------------------- run --

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attention": _own_attention, "store": _own_store, "read": _own_read, "shared": _own_shared}[kind](state)
    return {"attention": _plain_attention, "store": _plain_store, "read": _plain_read,
            "shared": _plain_shared}[kind](state)


def _own_batch(state, ops):
    news = [b - a for a, b in zip(state["start_host"], state["start_host"][1:])]
    return ops.PagedBatch(state["table"], state["lens"], state["start"], max_query=max(max(news), 1),
                          max_len=max(state["lens_host"]))


def _own_pages(pool, ops):
    return ops.QuantizedPages(*pool) if len(pool) == 2 else pool[0]


def _own_attention(state):
    from adaptiveimi_amd import ops

    case = state["case"]
    return ops.paged_attention(state["q"], _own_pages(state["k"], ops), _own_pages(state["v"], ops),
                               _own_batch(state, ops), window=case["window"], sinks=case["sinks"], out=state["out"],
                               lse=state["lse"])


def _own_store(state):
    from adaptiveimi_amd import ops

    case = state["case"]
    batch = _own_batch(state, ops)
    keys, values = _own_pages(state["key_pages"], ops), _own_pages(state["value_pages"], ops)
    q, _ = ops.qk_norm_rope(state["q"], state["k"], inv_freq=state["inv_freq"], query_weight=state["qw"],
                            key_weight=state["kw"], eps=EPS, interleaved=case["interleaved"],
                            query_out=state["q_out"], value=state["v"], batch=batch, key_pages=keys,
                            value_pages=values)
    shape = (len(state["lens_host"]), case["kv_heads"], state["rows"], case["dim"])
    k, v = torch.zeros(shape, dtype=q.dtype, device=DEV), torch.zeros(shape, dtype=q.dtype, device=DEV)
    return (q,) + ops.read_pages(keys, values, batch, first=state["first"], out=(k, v))


def _own_read(state):
    from adaptiveimi_amd import ops

    return ops.read_pages(_own_pages(state["k"], ops), _own_pages(state["v"], ops), _own_batch(state, ops),
                          out=(state["keys"], state["values"]))


def _own_shared(state):
    from adaptiveimi_amd import ops

    batch = ops.share_prefixes(_own_batch(state, ops), state["case"]["page"])
    return [ops.paged_attention(x["q"], _own_pages(x["k"], ops), _own_pages(x["v"], ops), batch, out=x["out"],
                                lse=x["lse"]) for x in state["layers"]]


# -------------------------------------------------------------- plain form --

def _rows(case, table, pool, s, n):
    """The first n rows of sequence s in 32 bits, [H, n, D]."""
    ids = table[s, :-(-n // case["page"])].long()
    parts = [t[ids].transpose(0, 1).flatten(1, 2)[:, :n] for t in pool]
    return _decode(*parts, case["fmt"]) if case["fmt"] else parts[0].float()


def _attend(case, state, q_all, k_pool, v_pool, out, lse, window=0, sinks=0):
    H, G, D = case["kv_heads"], case["groups"], case["dim"]
    scale = 1.0 / math.sqrt(D)
    for s, n in enumerate(state["lens_host"]):
        lo, hi = state["start_host"][s], state["start_host"][s + 1]
        if hi == lo:
            continue
        k, v = _rows(case, state["table"], k_pool, s, n), _rows(case, state["table"], v_pool, s, n)
        step = max(1, (1 << 28) // (H * G * n))   # scores of a gigabyte at most
        for a in range(lo, hi, step):
            b = min(hi, a + step)
            pos = torch.arange(n - hi + a, n - hi + b, device=DEV)
            first, last = n - hi + a, n - hi + b   # the keys that these rows can see
            lower = max(0, first - window + 1) if window else 0
            col = torch.arange(lower, last, device=DEV)
            ks, vs = k[:, lower:last], v[:, lower:last]
            if lower > 0 and sinks:
                head = min(sinks, lower)
                col = torch.cat([torch.arange(head, device=DEV), col])
                ks, vs = torch.cat([k[:, :head], ks], 1), torch.cat([v[:, :head], vs], 1)
            q = q_all[a:b].float().view(b - a, H, G, D).permute(1, 0, 2, 3).reshape(H, (b - a) * G, D)
            x = torch.matmul(q, ks.transpose(1, 2)) * scale
            seen = col[None] <= pos[:, None]
            if window:
                seen &= (col[None] > pos[:, None] - window) | (col[None] < sinks)
            x = x.view(H, b - a, G, -1).masked_fill_(~seen[None, :, None], -math.inf)
            top = x.amax(-1, keepdim=True)
            w = torch.exp(x - top)
            total = w.sum(-1, keepdim=True)
            o = torch.matmul(w.view(H, (b - a) * G, -1), vs).view(H, b - a, G, D) / total
            out[a:b] = o.permute(1, 0, 2, 3).reshape(b - a, H * G, D).to(out.dtype)
            lse[a:b] = (top + torch.log(total))[..., 0].permute(1, 0, 2).reshape(b - a, H * G)
    return out, lse


def _plain_attention(state):
    case = state["case"]
    return _attend(case, state, state["q"], state["k"], state["v"], state["out"], state["lse"], case["window"],
                   case["sinks"])


def _plain_shared(state):
    return [_attend(state["case"], state, x["q"], x["k"], x["v"], x["out"], x["lse"]) for x in state["layers"]]


def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    head, tail = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = head[..., :half], head[..., half:]
        head = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([head, tail], -1)


def _plain_store(state):
    case = state["case"]
    n = state["start_host"][-1]

    def one(x, w):
        x = x[:n].float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        if state["inv_freq"] is None:
            return x
        ang = state["positions"].double()[:, None] * state["inv_freq"].double()
        return _rotate(x, torch.cos(ang).float(), torch.sin(ang).float(), case["interleaved"])

    state["q_out"][:n] = one(state["q"], state["qw"]).to(state["q_out"].dtype)
    pages, slot = state["slots"]
    result = [state["q_out"]]
    seq = torch.repeat_interleave(torch.diff(state["start"]).long(), output_size=n)
    at = state["positions"] - state["first"][seq]
    for x, pool in ((one(state["k"], state["kw"]), state["key_pages"]), (state["v"][:n].float(), state["value_pages"])):
        codes, exps = _encode(x, case["fmt"])
        whole = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
        whole(pool[0])[pages, :, slot] = whole(codes)
        pool[1][pages, :, slot] = exps
        back = torch.zeros((len(state["lens_host"]), case["kv_heads"], state["rows"], case["dim"]),
                           dtype=state["q_out"].dtype, device=DEV)
        back[seq, :, at] = _decode(whole(pool[0])[pages, :, slot].view(codes.dtype), pool[1][pages, :, slot],
                                   case["fmt"]).to(back.dtype)
        result.append(back)
    return tuple(result)


def _plain_read(state):
    for pool, out in ((state["k"], state["keys"]), (state["v"], state["values"])):
        for s, n in enumerate(state["lens_host"]):
            out[s, :, :n] = _rows(state["case"], state["table"], pool, s, n).to(out.dtype)
    return state["keys"], state["values"]


# ------------------------------------------------------------------- exact --

def exact(case, seed):
    """The definition in 64 bits."""
    state = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(state, state["q"], state["k"], state["v"], case["window"], case["sinks"])
    if case["kind"] == "shared":
        return [_exact_attention(state, x["q"], x["k"], x["v"], 0, 0) for x in state["layers"]]
    return _exact_store(state) if case["kind"] == "store" else _exact_read(state)


def _power(k):
    """2^k in 64 bits, exactly (a power function need not be)."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _values64(case, pool):
    """A tensor of rows in 64 bits, read off the bits of its codes."""
    fmt = case["fmt"]
    if not fmt:
        return pool[0].double()
    codes, e = pool
    if fmt == "int8":
        x = codes.double()
    else:
        bits, lead = (codes.view(torch.uint8), 3) if fmt == "fp8" else (codes, 1)   # bits of the significand
        if fmt == "fp4":
            bits = torch.stack([bits % 16, bits // 16], -1).flatten(-2)
        bits = bits.long()
        sign = 1.0 - 2.0 * (bits >> (7 if fmt == "fp8" else 3)).double()
        power, m = (bits >> lead) & (15 if fmt == "fp8" else 3), (bits & ((1 << lead) - 1)).double() / (1 << lead)
        bias = 7 if fmt == "fp8" else 1
        x = sign * torch.where(power > 0, (1 + m) * _power(power - bias), m * 2.0 ** (1 - bias))
    return x * torch.repeat_interleave(_power(e.long() - 127), BLOCK, -1)


def _exact_attention(state, q, k_pool, v_pool, window, sinks):
    case = state["case"]
    H, G, D, page = case["kv_heads"], case["groups"], case["dim"], case["page"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    for s, n in enumerate(state["lens_host"]):
        lo, hi = state["start_host"][s], state["start_host"][s + 1]
        row = torch.arange(n, device=DEV)
        ids = state["table"][s].long()[row // page]
        for h in range(H):
            k = _values64(case, [t[ids, h, row % page] for t in k_pool])
            v = _values64(case, [t[ids, h, row % page] for t in v_pool])
            for a in range(lo, hi, 1024):
                b = min(hi, a + 1024)
                pos = (n - hi + torch.arange(a, b, device=DEV))[:, None]
                hidden = row[None] > pos
                if window:
                    hidden |= (row[None] <= pos - window) & (row[None] >= sinks)
                for g in range(h * G, h * G + G):
                    x = (q[a:b, g].double() @ k.T) / math.sqrt(D)
                    x[hidden] = -math.inf
                    lse[a:b, g] = torch.logsumexp(x, -1)
                    out[a:b, g] = torch.softmax(x, -1) @ v
    return out, lse


def _nearest(x, fmt):
    """What a quantised pool makes of values [..., dim]: to the nearest of the
    format's numbers, ties to the even code, times the block's power."""
    top = x.unflatten(-1, (-1, BLOCK)).abs().amax(-1)
    k = torch.ceil(torch.log2(top / LARGEST[fmt])).clamp(min=-117)
    k += (top > LARGEST[fmt] * _power(k)).double()   # where the logarithm was rounded
    k -= (top <= LARGEST[fmt] * _power(k - 1)).double()
    scale = torch.repeat_interleave(_power(k.clamp(min=-117)), BLOCK, -1)
    y = x / scale
    if fmt == "int8":
        step = torch.ones_like(y)
    else:   # the distance of neighbours in the binade of |y|
        low, bits = (-6, 3) if fmt == "fp8" else (0, 1)
        step = _power((torch.frexp(y)[1] - 1).clamp(min=low) - bits)
    return torch.round(y / step) * step * scale


def _exact_store(state):
    case = state["case"]
    n, r = state["start_host"][-1], case["rotary"]

    def one(x, w):
        y = x[:n].double()
        if w is not None:
            y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + EPS) * w.double()
        if r:
            turn = torch.polar(torch.ones((n, r // 2), dtype=torch.float64, device=DEV),
                               state["positions"].double()[:, None] * state["inv_freq"].double()[None])
            even, odd = ((slice(0, r, 2), slice(1, r, 2)) if case["interleaved"]
                         else (slice(0, r // 2), slice(r // 2, r)))
            z = torch.complex(y[..., even], y[..., odd]) * turn[:, None]
            y[..., even], y[..., odd] = z.real, z.imag
        return y

    q = state["q_out"].double()
    q[:n] = one(state["q"], state["qw"])
    result = [q]
    for x in (_nearest(one(state["k"], state["kw"]), case["fmt"]), _nearest(state["v"][:n].double(), case["fmt"])):
        back = torch.zeros((len(state["lens_host"]), case["kv_heads"], state["rows"], case["dim"]),
                           dtype=torch.float64, device=DEV)
        for s in range(len(state["lens_host"])):
            lo, hi = state["start_host"][s], state["start_host"][s + 1]
            back[s, :, :hi - lo] = x[lo:hi].transpose(0, 1)
        result.append(back)
    return tuple(result)


def _exact_read(state):
    case = state["case"]
    result = []
    for pool in (state["k"], state["v"]):
        out = state["keys"].double()
        for s, n in enumerate(state["lens_host"]):
            row = torch.arange(n, device=DEV)
            ids = state["table"][s].long()[row // case["page"]]
            for h in range(case["kv_heads"]):
                out[s, h, :n] = _values64(case, [t[ids, h, row % case["page"]] for t in pool])
        result.append(out)
    return tuple(result)


# -------------------------------------------------------------------- work --

def work(case):
    return {"attention": _work_attention, "store": _work_store, "read": _work_read,
            "shared": _work_shared}[case["kind"]](case)


def _row_bytes(case):
    """A row of one head in the pool."""
    D, fmt = case["dim"], case["fmt"]
    return 2 * D if not fmt else (D // 2 if fmt == "fp4" else D) + D // BLOCK


def _work_attention(case):
    H, G, D, window, sinks = case["kv_heads"], case["groups"], case["dim"], case["window"], case["sinks"]
    pairs = rows = tokens = 0
    for n, m in zip(_ints(case["lens"]), _ints(case["news"])):
        tokens += m
        first = n - m
        if not window:
            pairs += m * first + m * (m + 1) // 2
            rows += n
            continue
        for p in range(first, n):
            low = max(0, p - window + 1)
            pairs += p + 1 - low + min(sinks, low)
        low = max(0, first - window + 1)
        rows += n - low + min(sinks, low)
    return {"bytes": 4 * D * tokens * H * G + 2 * rows * H * _row_bytes(case) + 4 * tokens * H * G,
            "flops": 4 * D * H * G * pairs}


def _work_store(case):
    """Inputs read, queries written, rows written and, decoded, read back."""
    H, G, D = case["kv_heads"], case["groups"], case["dim"]
    tokens = sum(_ints(case["news"]))
    per = 2 * D * (2 * H * G + 2 * H) + 2 * H * (2 * _row_bytes(case) + 2 * D)
    return {"bytes": per * tokens, "flops": 8 * D * (H * G + H) * tokens}


def _work_read(case):
    rows = sum(_ints(case["lens"])) * case["kv_heads"] * 2
    return {"bytes": rows * (_row_bytes(case) + 2 * case["dim"]), "flops": rows * case["dim"]}


def _work_shared(case):
    """Shared rows read once for each prompt, own rows once."""
    H, G, D, new, page = case["kv_heads"], case["groups"], case["dim"], case["new"], case["page"]
    prompts, own_rows, width = _ints(case["prompts"]), _ints(case["own"]), case["width"]
    common = sum(p // page * page for p in prompts)
    rows = common + sum(own_rows) + sum(width * (p % page) for p in prompts)
    tokens = new * len(own_rows)
    pairs = sum(new * (prompts[i // width] + n) - new * (new - 1) // 2 for i, n in enumerate(own_rows))
    return {"bytes": case["layers"] * (4 * D * tokens * H * G + 2 * rows * H * _row_bytes(case) + 4 * tokens * H * G),
            "flops": case["layers"] * 4 * D * H * G * pairs}
