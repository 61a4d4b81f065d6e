"""Cases of the 8-bit key/value cache: writing it, reading it back, and the attention that reads it.

Rows of keys and values (the ``head_dim`` values of one position and kv head) are held as one byte a value and one byte
a row: the exponent of a power-of-two scale, plus 127. ``fp8`` rows hold e4m3 codes, ``int8`` rows codes from -127 to 127.
Pages hold 64 positions: codes ``[pages, kv_heads, 64, head_dim]``, exponents ``[pages, kv_heads, 64]``.

Kinds of cases:

* ``cache``: a step's keys and values into the cache, then the pages of the step's sequences read back;
* ``decode``: one new token per sequence attends over the cache;
* ``chunk``: several new tokens per sequence attend over the cache (which holds theirs already).
"""
import random

import torch

own = False

PAGE = 64
LARGEST = {"fp8": (1.75, 8), "int8": (1.984375, 6)}   # the largest code as m * 2^E
LEAST = -100                                           # the least exponent of a row's scale

# heads, kv heads, head size: the sizes of the benchmark's three models, then those of the tests' small ones
SIZES = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (6, 3, 64), (4, 2, 128), (3, 1, 32), (5, 5, 48)]


def _case(name, kind, sizes, fmt, seqs, longest, shortest, new, window=0, dtype="bfloat16"):
    heads, kv_heads, head_dim = sizes
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "fmt": fmt, "seqs": seqs,
         "longest": longest, "shortest": shortest, "new": new, "window": window, "dtype": dtype}
    return dict(c, name=name) if name else c


def listed():
    small, middle, large = SIZES[:3]
    return [
        # one short conversation, one token: what a user at the prompt waits for
        _case("decode_1x77", "decode", small, "fp8", 1, 77, 77, 1),
        # the benchmark's batch: eight sequences around 2,048 positions
        _case("decode_8x2060", "decode", small, "fp8", 8, 2060, 1900, 1),
        # a busy server: many sequences of unequal lengths, the more exact format
        _case("decode_64_ragged_int8", "decode", large, "int8", 64, 4000, 200, 1),
        # long contexts at the model's limit: the cache is most of what a step reads
        _case("decode_8x32768", "decode", large, "fp8", 8, 32768, 30000, 1),
        # a chat turn: a few tokens onto a live conversation
        _case("chunk_9_onto_1000", "chunk", small, "fp8", 1, 1009, 1009, 9),
        # sequences that decode and prompts that arrive, in one step, in windowed layers
        _case("chunk_mixed_window", "chunk", middle, "int8", 6, 3001, 300, 190, window=1000),
        # a portion of a long prompt
        _case("chunk_512_onto_8000", "chunk", small, "fp8", 1, 8512, 8512, 512),
        # a large portion of a document
        _case("chunk_1024_onto_16000", "chunk", large, "fp8", 1, 17024, 17024, 1024),
        # a decode step's keys and values, and a look at what the cache holds
        _case("cache_1_token", "cache", small, "fp8", 1, 40, 40, 1),
        _case("cache_8x1_int8", "cache", middle, "int8", 8, 700, 300, 1),
        # prompts of unequal lengths, in the true 32-bit path
        _case("cache_prompts_float", "cache", small, "int8", 5, 2000, 130, 2000, dtype="float32"),
        # long prompts
        _case("cache_prompts_long", "cache", large, "fp8", 8, 8192, 7000, 8192),
    ]


def draw(rng):
    kind = rng.choice(["decode", "chunk", "cache"])
    fmt = rng.choice(["fp8", "int8"])
    span = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))
    if kind == "cache":
        sizes, seqs, longest = rng.choice(SIZES), span(1, 48), span(1, 8192)
        while seqs * longest > 65536:
            seqs = max(1, seqs // 2)
        new = 1 if rng.random() < 0.3 else span(1, longest)
        return _case("", kind, sizes, fmt, seqs, longest, span(max(1, longest // 8), longest), new, 0,
                     rng.choice(["bfloat16", "bfloat16", "float32"]))
    if kind == "decode":
        sizes, seqs, longest = rng.choice(SIZES), span(1, 96), span(1, 32768)
        while seqs * longest > 262144:
            seqs = max(1, seqs // 2)
        window = span(16, 4096) if rng.random() < 0.2 else 0
        return _case("", kind, sizes, fmt, seqs, longest, span(max(1, longest // 8), longest), 1, window)
    sizes, seqs = rng.choice(SIZES[:5]), span(1, 8)
    new = span(2, 1024)
    longest = new + span(1, 15000)
    while seqs * new * longest > 1024 * 16000:
        seqs, new, longest = max(1, seqs // 2), new - new // 4, longest - (longest - new) // 4
    window = span(64, 4096) if rng.random() < 0.2 else 0
    return _case("", kind, sizes, fmt, seqs, longest, span(max(1, longest // 8), longest), new, window)


def _lengths(case):
    """Per sequence: its length before the step, and its new tokens. The first sequence is the longest and brings the
    most; what the others are goes by the case alone."""
    rng = random.Random(case["seqs"] * 1000003 + case["longest"] * 7919 + case["new"])
    ends, news = [case["longest"]], [case["new"]]
    for _ in range(case["seqs"] - 1):
        ends.append(rng.randint(case["shortest"], case["longest"]))
        news.append(case["new"] if case["new"] == 1 else rng.randint(1, case["new"]))
    news = [min(n, e) for n, e in zip(news, ends)]
    return [e - n for e, n in zip(ends, news)], news


def _pages(n):
    return -(-n // PAGE)


# ---- the format --------------------------------------------------------------------------------------------------------

def _power(e):
    """2^e as a float, from its bits (exact)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x, fmt):
    """Codes and exponents of rows of float values."""
    m, power = LARGEST[fmt]
    amax = x.abs().amax(-1)
    fraction, exponent = torch.frexp(amax)                # amax = (2 * fraction) * 2^(exponent - 1)
    e = (exponent - 1 - power + (2 * fraction > m)).clamp(min=LEAST)
    e = torch.where(amax > 0, e, torch.full_like(e, LEAST))
    y = x * _power(-e).unsqueeze(-1)
    codes = y.to(torch.float8_e4m3fn) if fmt == "fp8" else torch.round(y).to(torch.int8)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, scale):
    return codes.float() * _power(scale.int() - 127).unsqueeze(-1)


# ---- what a program has before the call --------------------------------------------------------------------------------

def _rows(g, shape, device):
    """Keys or values as a layer gives them: normal, with rows (positions) and columns (dimensions) of unequal size."""
    x = torch.randn(shape, generator=g, device=device)
    x *= torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device=device))
    return x.mul_(torch.exp(0.7 * torch.randn(shape[-1:], generator=g, device=device)))


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    starts, news = _lengths(case)
    S, kvh, hd = case["seqs"], case["kv_heads"], case["head_dim"]
    ends = [s + n for s, n in zip(starts, news)]
    counts = [_pages(e) for e in ends]
    most, total, T = max(counts), sum(counts) + 3, sum(news)
    # the pages lie in no order, as after many requests
    order = torch.randperm(total, generator=g, device=device).to(torch.int32)
    table = torch.zeros((S, most), dtype=torch.int32)
    first = 0
    order_host = order.tolist()
    for i, n in enumerate(counts):
        table[i, :n] = torch.tensor(order_host[first:first + n], dtype=torch.int32)
        first += n
    state = {"case": case, "table": table.to(device), "most": most, "longest": max(ends), "scale": hd ** -0.5}
    seq_of = torch.repeat_interleave(torch.arange(S), torch.tensor(news))
    cu = torch.tensor([0] + news).cumsum(0)
    place = torch.arange(T) - cu[seq_of]                   # a token's place among its sequence's new ones
    positions = torch.tensor(starts)[seq_of] + place
    state["positions"], state["seq_of"], state["place"] = (t.to(device) for t in (positions, seq_of, place))
    state["ends"] = torch.tensor(ends, device=device)
    state["news"] = news
    for which in ("k", "v"):
        x = _rows(g, (total, kvh, PAGE, hd), device)
        state[which + "_codes"], state[which + "_scale"] = _quantise(x, case["fmt"])
        del x
    if case["kind"] == "cache":
        state["k"] = _rows(g, (T, kvh, hd), device).to(dtype)
        state["v"] = _rows(g, (T, kvh, hd), device).to(dtype)
    else:
        state["q"] = (torch.randn((T, case["heads"], hd), generator=g, device=device) * 1.5).to(dtype)
    if own:   # the step and the cache as the engine hands them to its layers
        from smolmoe_c99_b200.cache import LayerCache
        from smolmoe_c99_b200.engine.batch import pack_step
        state["step"] = pack_step(list(range(S)), starts, [[0] * n for n in news], device)
        state["layer"] = LayerCache("kv", state["k_codes"], state["v_codes"], state["table"], 0, case["window"] or None,
                                    k_scale=state["k_scale"], v_scale=state["v_scale"])
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------

def _gather(state, which):
    """The pages of the step's sequences as float values: [sequences, pages, kv heads, 64, head size]."""
    pages = state["table"].long()
    codes = state[which + "_codes"]
    codes = codes.view(torch.uint8)[pages].view(codes.dtype)
    return _values(codes, state[which + "_scale"][pages])


def _plain_cache(state):
    case = state["case"]
    dtype = getattr(torch, case["dtype"])
    page = state["table"][state["seq_of"], state["positions"] // PAGE].long()
    at = state["positions"] % PAGE
    out = []
    for which in ("k", "v"):
        codes, scale = _quantise(state[which].float(), case["fmt"])
        state[which + "_codes"].view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
        state[which + "_scale"][page, :, at] = scale
        x = _gather(state, which)
        here = torch.arange(state["most"] * PAGE, device=x.device).view(1, state["most"], 1, PAGE, 1)
        out.append(torch.where(here < state["ends"].view(-1, 1, 1, 1, 1), x, torch.zeros((), device=x.device)).to(dtype))
    return out


def _plain_attention(state):
    case = state["case"]
    S, H, G, hd = case["seqs"], case["heads"], case["kv_heads"], case["head_dim"]
    L, N = state["most"] * PAGE, max(state["news"])
    q = state["q"].float()
    padded = torch.zeros((S, N, H, hd), device=q.device)
    padded[state["seq_of"], state["place"]] = q
    pos = torch.full((S, N), -1, dtype=torch.long, device=q.device)
    pos[state["seq_of"], state["place"]] = state["positions"]
    # per kv head the rows are (new token, head of the group)
    qs = padded.view(S, N, G, H // G, hd).permute(0, 2, 1, 3, 4).reshape(S, G, N * (H // G), hd)
    k = _gather(state, "k").permute(0, 2, 1, 3, 4).reshape(S, G, L, hd)
    s = torch.matmul(qs, k.transpose(-1, -2)).mul_(state["scale"]).view(S, G, N, H // G, L)
    del k
    key = torch.arange(L, device=q.device)
    seen = key <= pos.unsqueeze(-1)
    if case["window"]:
        seen &= key > pos.unsqueeze(-1) - case["window"]
    s.masked_fill_(~seen.view(S, 1, N, 1, L), float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top > float("-inf"), top, torch.zeros((), device=q.device))))
    v = _gather(state, "v").permute(0, 2, 1, 3, 4).reshape(S, G, L, hd)
    # what lies behind a sequence's end is no part of it
    v = torch.where((key < state["ends"].view(-1, 1)).view(S, 1, L, 1), v, torch.zeros((), device=q.device))
    o = torch.matmul(p.view(S, G, N * (H // G), L), v).view(S, G, N, H // G, hd) / p.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3, 4).reshape(S, N, H, hd)
    return o[state["seq_of"], state["place"]].to(state["q"].dtype)


def run(state):
    case = state["case"]
    if own:
        from smolmoe_c99_b200.kernels import get_ops
        ops = get_ops()
        if case["kind"] == "cache":
            ops.kv_quant_store(state["k"], state["v"], state["step"], state["layer"])
            pages = ops.kv_quant_load(state["step"], state["layer"], state["k"].dtype)
            shape = (case["seqs"], state["most"], case["kv_heads"], PAGE, case["head_dim"])
            return [pages.k_pool.view(shape), pages.v_pool.view(shape)]
        return ops.attention_quant(state["q"], state["step"], state["scale"], case["window"], state["layer"])
    return _plain_cache(state) if case["kind"] == "cache" else _plain_attention(state)


# ---- the least a pass reads, writes and computes -----------------------------------------------------------------------

def work(case):
    starts, news = _lengths(case)
    heads, kvh, hd, window = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    size = 4 if case["dtype"] == "float32" else 2
    row = kvh * 2 * (hd + 1)                               # bytes of a position in the cache
    if case["kind"] == "cache":
        ends = [s + n for s, n in zip(starts, news)]
        padded = case["seqs"] * max(_pages(e) for e in ends) * PAGE
        return {"bytes": sum(news) * (kvh * 2 * hd * size + row) + sum(ends) * row + padded * kvh * 2 * hd * size, "flops": 0}
    read, pairs = 0, 0
    for s, n in zip(starts, news):
        read += s + n - (max(0, s - window + 1) if window else 0)
        if window:
            pairs += sum(min(p + 1, window) for p in range(s, s + n))
        else:
            pairs += n * s + n * (n + 1) // 2
    return {"bytes": read * row + 2 * sum(news) * heads * hd * size, "flops": 4 * hd * heads * pairs}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------

def _exact_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rows(x, fmt):
    """What the cache stands for where it was given the rows ``x``: each value to the nearest of its row's grid."""
    x = x.double()
    top = {"fp8": 448.0, "int8": 127.0}[fmt]
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / top))
    e = torch.where(amax > top * _exact_power(e), e + 1, torch.where(amax <= top * _exact_power(e - 1), e - 1, e))
    e = torch.where(amax > 0, e, torch.full_like(e, LEAST)).clamp(min=LEAST)
    y = x / _exact_power(e)
    if fmt == "fp8":     # three bits behind the leading one, from 2^-6 on; steps of 2^-9 below
        lead = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
        lead = torch.where(_exact_power(lead + 1) <= y.abs(), lead + 1, lead)
        step = _exact_power(lead - 3)
    else:
        step = torch.ones_like(y)
    return torch.round(y / step) * step * _exact_power(e)


def _exact_sequence(state, which, i, length):
    """The first ``length`` positions of sequence ``i`` from the cache: [kv heads, length, head size] in 64 bits."""
    pages = state["table"][i, :_pages(length)].long()
    codes, scale = state[which + "_codes"], state[which + "_scale"]
    x = codes.view(torch.uint8)[pages].view(codes.dtype).double() * _exact_power(scale[pages].long() - 127).unsqueeze(-1)
    return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[-1])[:, :length]


def exact(case, seed):
    state = prepare(case, seed)
    starts, news = _lengths(case)
    kvh, hd, group = case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    if case["kind"] == "cache":
        out = []
        for which in ("k", "v"):
            rows = _exact_rows(state[which], case["fmt"])
            pages = torch.zeros((case["seqs"], state["most"], kvh, PAGE, hd), dtype=torch.float64, device=rows.device)
            first = 0
            for i, (s, n) in enumerate(zip(starts, news)):
                flat = torch.zeros((kvh, state["most"] * PAGE, hd), dtype=torch.float64, device=rows.device)
                if s:
                    flat[:, :s] = _exact_sequence(state, which, i, s)
                flat[:, s:s + n] = rows[first:first + n].transpose(0, 1)
                pages[i] = flat.view(kvh, state["most"], PAGE, hd).transpose(0, 1)
                first += n
            out.append(pages)
        return out
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    first = 0
    for i, (s, n) in enumerate(zip(starts, news)):
        k, v = (_exact_sequence(state, which, i, s + n) for which in ("k", "v"))
        q = state["q"][first:first + n].double()
        rows, keys = torch.arange(s, s + n, device=q.device).view(-1, 1), torch.arange(s + n, device=q.device)
        hidden = (keys > rows) | ((keys <= rows - case["window"]) if case["window"] else torch.zeros_like(keys, dtype=torch.bool))
        for h in range(case["heads"]):
            x = (q[:, h] @ k[h // group].T) * state["scale"]
            x[hidden] = float("-inf")
            out[first:first + n, h] = torch.softmax(x, -1) @ v[h // group]
        first += n
    return out
