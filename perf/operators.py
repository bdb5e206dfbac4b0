"""Cases of the operators for int8 decoder layers: per-token quantisation, the
scaled int8 product, and the quantised K/V cache (append, read, attention).

Every case is one pass through one operator as a serving program calls it.
``own`` selects the framework's kernels; otherwise ``run`` computes the same
operators from elementary torch operations.

Definitions (L = 2^bits - 1; rte = round half to even; quotients are exact
before they are rounded, so codes do not depend on who computes them):

* per token:  s = f32(max|x| / 127), q = clamp(rte(x / s), -127, 127)
* product:    out = (q @ w) * s_token * s_channel [+ bias] [+ residual]
* cache, per (token, head, group of dims):  lo = bf16 rounded down (min x),
  s = bf16 rounded up ((max x - lo) / L), c = clamp(rte((x - lo) / s), 0, L);
  the cache stands for the values c * s + lo
* attention:  token i of the n new tokens of a sequence of length len stands
  at position len - n + i and attends to every position up to its own.
"""

import math
import random

import torch

own = False

DEV = "cuda:0"
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_BF16_MAX = 3.3895313892515355e38


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one token entering a layer of this repository's encoder width: all latency
        dict(name="quantize_token", op="quantize", tokens=1, width=768, dtype="bf16"),
        # the activations of a long prompt chunk before a feed-forward projection
        dict(name="quantize_chunk", op="quantize", tokens=8192, width=8192, dtype="bf16"),
        # a few sequences decoding: the whole weight is read for four tokens
        dict(name="product_decode", op="product", tokens=4, k=4096, n=4096, out="bf16",
             bias=False, residual=False),
        # a ragged prompt through a projection with bias and residual, fp32 out
        dict(name="product_ragged", op="product", tokens=777, k=768, n=2311, out="f32",
             bias=True, residual=True),
        # a long prompt chunk through a wide feed-forward projection
        dict(name="product_prompt", op="product", tokens=8192, k=4096, n=14336, out="bf16",
             bias=False, residual=False),
        # one decode step of a batch writes its tokens into a 4-bit cache
        dict(name="append_decode", op="append", batch=64, length=4001, new=1, kv_heads=8, dim=128,
             bits=4, group=64, page=64, dtype="bf16"),
        # ragged prompts written into an 8-bit cache of small pages
        dict(name="append_prompt", op="append", batch=7, length=3001, new=3001, kv_heads=8, dim=128,
             bits=8, group=64, page=16, dtype="f16"),
        # the newest tokens of a few sequences read back in fp32
        dict(name="read_recent", op="read", batch=5, length=300, new=33, kv_heads=12, dim=64,
             bits=8, group=32, page=32, dtype="f32"),
        # whole sequences read back from a 4-bit cache: a prefix to be reused
        dict(name="read_prefix", op="read", batch=6, length=8100, new=8100, kv_heads=8, dim=128,
             bits=4, group=64, page=64, dtype="bf16"),
        # one short sequence decoding, a K/V head for every query head: latency
        dict(name="attend_short", op="attend", batch=1, length=500, new=1, kv_heads=12, share=1,
             dim=64, bits=8, group=32, page=16, dtype="f32"),
        # a ragged batch decoding over long contexts with shared K/V heads
        dict(name="attend_batch", op="attend", batch=64, length=16000, new=1, kv_heads=8, share=4,
             dim=128, bits=4, group=64, page=64, dtype="bf16"),
        # prompt chunks attending to their cached prefix and to themselves
        dict(name="attend_chunk", op="attend", batch=2, length=6000, new=1024, kv_heads=8, share=4,
             dim=128, bits=4, group=64, page=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _size(rng, lo, hi, step):
    """Over the logarithm; a multiple of ``step`` two times in three, else as it falls."""
    n = _log(rng, lo, hi)
    return max(step, n // step * step) if rng.random() < 0.67 else n


_TOKEN_HEADS = 64 * 16000 * 8 * 128 * 5 // 8      # cache elements of the largest case
_ATTEND_MACS = 2 * 1024 * 32 * 6000 * 128         # products of the largest case


def draw(rng):
    op = rng.choice(["quantize", "product", "append", "read", "attend", "attend"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "quantize":
        tokens, width = _size(rng, 1, 8192, 8), _size(rng, 64, 8192, 64)
        return dict(op=op, tokens=tokens, width=width, dtype=dtype)
    if op == "product":
        k, n = _size(rng, 64, 8192, 64), _size(rng, 64, 14336, 64)
        tokens = _size(rng, 1, 8192, 8)
        while tokens * k * n > 8192 * 4096 * 14336:
            tokens //= 2
        return dict(op=op, tokens=tokens, k=k, n=n, out=dtype, bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5)
    case = dict(op=op, batch=_log(rng, 1, 128), length=_log(rng, 1, 16000), new=1,
                kv_heads=_log(rng, 1, 16))
    if op == "attend":
        case["share"] = rng.choice([1, 2, 3, 4, 5, 7, 8])
    case.update(dim=rng.choice([64, 128, 256]), bits=rng.choice([4, 8]), group=rng.choice([32, 64]),
                page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype)
    while case["batch"] * case["length"] * case["kv_heads"] * case["dim"] > _TOKEN_HEADS:
        case["batch"], case["length"] = (case["batch"] + 1) // 2, (case["length"] + 1) // 2
    kind = rng.choice(["one", "few", "chunk"])
    if kind == "few":
        case["new"] = _log(rng, 2, 16)
    elif kind == "chunk":
        case["new"] = _log(rng, 17, 2048) if op == "attend" else case["length"]
    case["new"] = min(case["new"], case["length"])
    if op == "attend":
        while (case["batch"] * case["new"] * case["kv_heads"] * case["share"] * case["length"]
               * case["dim"] > _ATTEND_MACS):
            case["new"] = (case["new"] + 1) // 2
            if case["new"] == 1:
                break
    return case


def _lengths(case):
    """Ragged lengths and counts of new tokens; they belong to the case, not to the seed."""
    rng = random.Random(f"{case['batch']} {case['length']} {case['new']} {case['page']}")
    lens = [case["length"]]
    while len(lens) < case["batch"]:
        lens.append(max(1, round(case["length"] * rng.uniform(0.25, 1.0))))
    news = []
    for n in lens:
        if case["new"] == case["length"]:
            news.append(n)
        else:
            news.append(min(n, max(1, round(case["new"] * rng.uniform(0.5, 1.0)))))
    news[0] = min(case["new"], lens[0])
    return lens, news


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "quantize":
        t, w = case["tokens"], case["width"]
        return {"bytes": t * w * (_BYTES[case["dtype"]] + 1) + 4 * t, "flops": 2 * t * w}
    if case["op"] == "product":
        t, k, n, e = case["tokens"], case["k"], case["n"], _BYTES[case["out"]]
        b = t * k + k * n + 4 * t + 4 * n + t * n * e
        return {"bytes": b + 4 * n * case["bias"] + t * n * e * case["residual"], "flops": 2 * t * k * n}
    lens, news = _lengths(case)
    h, d, e = case["kv_heads"], case["dim"], _BYTES[case["dtype"]]
    token = 2 * h * (d * case["bits"] // 8 + 4 * d // case["group"])   # K and V of a cached token
    if case["op"] == "append":   # reads the token, writes the cache and the values it stands for
        return {"bytes": sum(news) * (token + 4 * h * d * e), "flops": sum(news) * 4 * h * d}
    if case["op"] == "read":
        return {"bytes": sum(news) * (token + 2 * h * d * e), "flops": sum(news) * 4 * h * d}
    hq = h * case["share"]
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for m, n in zip(lens, news))
    return {"bytes": sum(lens) * token + sum(news) * 2 * hq * d * e, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _activations(tokens, width, dtype, g):
    """Unit normal with a few strong channels and tokens of different strength."""
    x = torch.randn(tokens, width, generator=g, device=DEV)
    x *= 1 + 15 * (torch.rand(width, generator=g, device=DEV) < 0.004)
    x *= torch.exp(0.5 * torch.randn(tokens, 1, generator=g, device=DEV))
    return x.to(dtype)


def _keys_values(case, tokens, g):
    """K with channels of unequal strength and offset, V near unit normal."""
    h, d, dt = case["kv_heads"], case["dim"], _DTYPES[case["dtype"]]
    k = torch.randn(tokens, h, d, generator=g, device=DEV, dtype=dt)
    k *= torch.exp(0.5 * torch.randn(h, d, generator=g, device=DEV)).to(dt)
    k += torch.randn(h, d, generator=g, device=DEV).to(dt)
    return k, torch.randn(tokens, h, d, generator=g, device=DEV, dtype=dt)


def _cumulative(counts):
    total = [0]
    for c in counts:
        total.append(total[-1] + c)
    return total


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "quantize":
        return dict(case=case, x=_activations(case["tokens"], case["width"], _DTYPES[case["dtype"]], g))
    if case["op"] == "product":
        state = _product_inputs(case, g)
        if own:   # the weight is laid out once, as a program does when it loads a model
            from iconnx_b200 import ops
            state["w"] = ops.prepare_weight(state["w"])
        return state
    return _prepare_cache(case, g, seed)


def _product_inputs(case, g):
    t, k, n, dt = case["tokens"], case["k"], case["n"], _DTYPES[case["out"]]
    x = _activations(t, k, torch.float32, g)
    q_scale = x.abs().amax(1) / 127
    q = torch.round(x / q_scale[:, None]).clamp(-127, 127).to(torch.int8)
    w = torch.randint(-127, 128, (k, n), generator=g, device=DEV, dtype=torch.int8)
    return dict(case=case, q=q, q_scale=q_scale, w=w,
                w_scale=(0.5 + torch.rand(n, generator=g, device=DEV)) / (73 * math.sqrt(k)),
                bias=torch.randn(n, generator=g, device=DEV) if case["bias"] else None,
                residual=(torch.randn(t, n, generator=g, device=DEV).to(dt)
                          if case["residual"] else None))


def _prepare_cache(case, g, seed):
    lens, news = _lengths(case)
    order = list(range(len(lens)))
    random.Random(seed).shuffle(order)
    lens, news = [lens[i] for i in order], [news[i] for i in order]
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    perm = torch.randperm(pool, generator=g, device=DEV).tolist()
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([perm.pop() for _ in range(n)], dtype=torch.int32)
    table = table.to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    state = dict(case=case, lens=lens, news=news, table=table, seq_lens=torch.tensor(lens, **i32),
                 cu=torch.tensor(_cumulative(news), **i32), tokens=sum(news))
    k, v = _keys_values(case, sum(news if case["op"] == "append" else lens), g)
    if own:
        from iconnx_b200 import kv_cache
        state["cache"] = kv_cache.KvCache(pool, page, h, d, bits=case["bits"], group=case["group"],
                                          device=DEV)
    else:
        state["cache"] = [_empty_plain(pool, page, h, d, case["group"]) for _ in range(2)]
    if case["op"] == "append":
        state.update(k=k, v=v)
        return state
    full = torch.tensor(_cumulative(lens), **i32)
    if own:
        kv_cache.gpu_kv_cache_append(state["cache"], k, v, table, state["seq_lens"], full)
    else:
        for plain, x in zip(state["cache"], (k, v)):
            for b, n in enumerate(lens):
                a = sum(lens[:b])
                slots = _slots(table, state["seq_lens"], full, page, a, a + n)
                _store_plain(plain, x[a:a + n], slots, case["bits"], case["group"])
    if case["op"] == "attend":
        hq = h * case["share"]
        state["q"] = torch.randn(state["tokens"], hq, d, generator=g, device=DEV).to(_DTYPES[case["dtype"]])
    return state


# -------------------------------------------------------------- plain form
def _round_bf16(x, up):
    """x (64 bits) rounded up or down to bf16."""
    b = x.to(torch.bfloat16)
    wrong = (b.double() < x) if up else (b.double() > x)
    bits = b.view(torch.int16)
    away = torch.where(b > 0, 1, -1) if up else torch.where(b > 0, -1, 1)
    step = torch.where(b == 0, torch.full_like(bits, 1 if up else -32767), bits + away.to(torch.int16))
    return torch.where(wrong, step, bits).view(torch.bfloat16)


def _codes(x, bits, group):
    """Codes [t, h, d] and per-group scale and low end [t, h, d / group]."""
    t, h, d = x.shape
    levels = (1 << bits) - 1
    x = x.reshape(t, h, d // group, group).double()
    low = _round_bf16(x.amin(-1), up=False).double().clamp(min=-_BF16_MAX)
    scale = _round_bf16((x.amax(-1) - low) / levels, up=True)
    s = scale.double()[..., None]
    c = torch.round((x - low[..., None]) / torch.where(s > 0, s, 1.0)).clamp(0, levels)
    return torch.where(s > 0, c, 0.0).to(torch.uint8).reshape(t, h, d), scale, low.to(torch.bfloat16)


def _values(codes, scale, low, group):
    t, h, d = codes.shape
    c = codes.reshape(t, h, d // group, group).float()
    return (c * scale.float()[..., None] + low.float()[..., None]).reshape(t, h, d)


def _empty_plain(pool, page, h, d, group):
    return dict(codes=torch.zeros(pool * page, h, d, dtype=torch.uint8, device=DEV),
                scale=torch.zeros(pool * page, h, d // group, dtype=torch.bfloat16, device=DEV),
                low=torch.zeros(pool * page, h, d // group, dtype=torch.bfloat16, device=DEV))


def _slots(table, seq_lens, cu, page, first, last):
    """Where the packed new tokens first..last-1 stand in the pool."""
    i = torch.arange(first, last, device=DEV)
    seq = (i[:, None] >= cu[None, 1:]).sum(1)
    pos = seq_lens[seq] - cu[seq + 1] + i
    return table[seq, pos // page].long() * page + pos % page


def _store_plain(plain, x, slots, bits, group):
    codes, scale, low = _codes(x, bits, group)
    plain["codes"][slots], plain["scale"][slots], plain["low"][slots] = codes, scale, low
    return _values(codes, scale, low, group)


def _load_plain(plain, slots, group):
    return _values(plain["codes"][slots], plain["scale"][slots], plain["low"][slots], group)


def _quantize_plain(x):
    x = x.double()
    scale = (x.abs().amax(1) / 127).float()
    s = scale.double()[:, None]
    q = torch.round(x / torch.where(s > 0, s, 1.0)).clamp(-127, 127)
    return torch.where(s > 0, q, 0.0).to(torch.int8), scale


def _product_plain(s):
    k = s["q"].shape[1]
    acc = None
    for a in range(0, k, 1024):    # 1024 products of 127 * 127 stay exact in 32-bit floats
        part = torch.matmul(s["q"][:, a:a + 1024].float(), s["w"][a:a + 1024].float()).int()
        acc = part if acc is None else acc + part
    out = acc.float() * s["q_scale"][:, None] * s["w_scale"][None]
    if s["bias"] is not None:
        out = out + s["bias"]
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(_DTYPES[s["case"]["out"]])


def _attend_plain(s):
    case = s["case"]
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    out = torch.empty_like(s["q"])
    a = 0
    for b, (n, new) in enumerate(zip(s["lens"], s["news"])):
        pos = torch.arange(n, device=DEV)
        slots = s["table"][b][pos // page].long() * page + pos % page
        k, v = (_load_plain(p, slots, case["group"]).transpose(0, 1) for p in s["cache"])
        q = s["q"][a:a + new].float().reshape(new, h, -1, d).permute(1, 2, 0, 3).reshape(h, -1, d)
        score = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(d)
        score = score.reshape(h, -1, new, n)
        if new > 1:
            score = score.masked_fill(pos[None] > pos[n - new:, None], -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).reshape(h, -1, n)
        o = torch.matmul(p, v).reshape(h, -1, new, d).permute(2, 0, 1, 3).reshape(new, -1, d)
        out[a:a + new] = o.to(out.dtype)
        a += new
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(s):
    case = s["case"]
    if case["op"] == "quantize":
        return _quantize_plain(s["x"])
    if case["op"] == "product":
        return _product_plain(s)
    if case["op"] == "attend":
        return _attend_plain(s)
    slots = _slots(s["table"], s["seq_lens"], s["cu"], case["page"], 0, s["tokens"])
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "append":
        return [_store_plain(p, x, slots, case["bits"], case["group"]).to(dt)
                for p, x in zip(s["cache"], (s["k"], s["v"]))]
    return [_load_plain(p, slots, case["group"]).to(dt) for p in s["cache"]]


# ------------------------------------------------------------ the framework
def _run_own(s):
    from iconnx_b200 import kv_cache, ops

    case = s["case"]
    if case["op"] == "quantize":
        return ops.gpu_quantize_per_token(s["x"])
    if case["op"] == "product":
        return ops.gpu_matmul_integer_scaled(s["q"], s["q_scale"], s["w"], s["w_scale"], bias=s["bias"],
                                             residual=s["residual"], out_dtype=_DTYPES[case["out"]])
    # one new token per sequence is the default; longer runs name their ends
    cu = None if s["tokens"] == case["batch"] else s["cu"]
    where = (s["table"], s["seq_lens"], cu)
    if case["op"] == "append":
        return kv_cache.gpu_kv_cache_append(s["cache"], s["k"], s["v"], *where, return_values=True)
    if case["op"] == "read":
        return kv_cache.gpu_kv_cache_read(s["cache"], *where, tokens=s["tokens"], dtype=_DTYPES[case["dtype"]])
    return kv_cache.gpu_kv_cache_attention(s["cache"], s["q"], *where)


# ------------------------------------------------------------------- exact
def _exact_bf16(x, up):
    """x rounded up or down to bf16, by its exponent in 64 bits."""
    exponent = torch.frexp(x)[1].clamp(min=-125).long()
    unit = ((exponent - 8 + 1023) << 52).view(torch.float64)   # 2^(exponent - 8), built exactly
    return (torch.ceil(x / unit) if up else torch.floor(x / unit)) * unit


def _exact_cached(x, bits, group):
    """What the cache stands for after x was written, in 64 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    top = 2 ** bits - 1
    for a in range(0, x.shape[0], 8192):
        for j in range(0, x.shape[2], group):
            part = x[a:a + 8192, :, j:j + group].double()
            low = _exact_bf16(part.min(-1, keepdim=True).values, up=False)
            step = _exact_bf16((part.max(-1, keepdim=True).values - low) / top, up=True)
            code = torch.where(step > 0, ((part - low) / step).round(), torch.zeros_like(part))
            out[a:a + 8192, :, j:j + group] = low + step * code.clamp(0, top)
    return out


def exact(case, seed):
    g = _gen(seed)
    if case["op"] == "quantize":
        x = _activations(case["tokens"], case["width"], _DTYPES[case["dtype"]], g)
        peak = x.double().abs().max(1).values
        step = (peak / 127).to(torch.float32).double()
        q = x.double().div(step[:, None]).round().clamp(-127, 127).nan_to_num(0.0)
        return q.to(torch.int8), peak / 127
    if case["op"] == "product":
        s = _product_inputs(case, g)
        out = torch.mm(s["q"].double() * s["q_scale"].double()[:, None],
                       s["w"].double() * s["w_scale"].double())
        for extra in (s["bias"], s["residual"]):
            if extra is not None:
                out += extra.double()
        return out
    return _exact_cache(case, seed)


def _exact_cache(case, seed):
    g = _gen(seed)
    lens, news = _lengths(case)
    order = list(range(len(lens)))
    random.Random(seed).shuffle(order)
    lens, news = [lens[i] for i in order], [news[i] for i in order]
    page = case["page"]
    torch.randperm(sum(-(-n // page) for n in lens) + 3, generator=g, device=DEV)   # the pages' order
    stored = news if case["op"] == "append" else lens
    k, v = _keys_values(case, sum(stored), g)
    if case["op"] == "append":
        return [_exact_cached(x, case["bits"], case["group"]) for x in (k, v)]
    ends = _cumulative(lens)
    if case["op"] == "read":
        return [torch.cat([_exact_cached(x[ends[b + 1] - news[b]:ends[b + 1]], case["bits"], case["group"])
                           for b in range(len(lens))]) for x in (k, v)]
    h, d, share = case["kv_heads"], case["dim"], case["share"]
    q = torch.randn(sum(news), h * share, d, generator=g, device=DEV).to(_DTYPES[case["dtype"]]).double()
    out = torch.empty_like(q)
    a = 0
    for b, new in enumerate(news):
        kb, vb = (_exact_cached(x[ends[b]:ends[b + 1]], case["bits"], case["group"]) for x in (k, v))
        hidden = torch.ones(new, lens[b], dtype=torch.bool, device=DEV).triu(lens[b] - new + 1)
        for i in range(h * share):
            logits = (q[a:a + new, i] @ kb[:, i // share].T) * d ** -0.5
            weights = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
            out[a:a + new, i] = weights @ vb[:, i // share]
        a += new
    return out
