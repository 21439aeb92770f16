"""Cases, inputs and plain forms of the operators of the 4-bit paged KV cache: append, attend, evict, read.

The cache.  A page holds 64 tokens of one stream; ``pool[layer, page]`` is ``kv_heads`` slabs of
``64 * (head_dim + head_dim / 16)`` bytes: K codes, V codes, K scales, V scales.  Thirty-two consecutive dims of one (token,
head) share a scale 2^(b - 127); a value is a 4-bit e2m1 code times it.  ``_fold`` / ``_unfold`` below are the byte order.

A batch is (seq_start, streams, ctx): sequence i owns rows seq_start[i] .. seq_start[i + 1] - 1, which are the entries
ctx[i] - n_i .. ctx[i] - 1 of its stream.  Row j of n attends to the ctx - n + j + 1 entries up to its own.
"""
import math

import torch

own = False

PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


# ---------------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one request without guidance, at the benchmark job's mean context: latency
        _attend("attend_single", 1, 1, 443, 443, 16, 16, 64, "bf16", False),
        # a full decode step of 32 guided requests (two streams each), contexts as the job holds them
        _attend("attend_batch", 64, 1, 120, 1000, 16, 16, 64, "bf16", False),
        # the same step with the weights that eviction needs, contexts past the first page table
        _attend("attend_batch_weights", 64, 1, 300, 2000, 16, 16, 64, "bf16", True),
        # long documents on shared key heads: what four bits are for
        _attend("attend_long_gqa", 16, 1, 9000, 32749, 32, 8, 128, "fp16", False),
        # five drafted tokens per request checked at once, with weights
        _attend("attend_draft_weights", 9, 5, 700, 6000, 24, 3, 128, "bf16", True),
        # prompts of the repository's lengths (34 conditioning rows + text, 513 the longest), with weights
        _attend("attend_prompt_weights", 6, 513, 513, 513, 16, 16, 64, "bf16", True),
        # a long prompt's chunk behind an earlier one, shared key heads
        _attend("attend_prompt_long", 2, 4095, 4700, 5001, 32, 8, 128, "bf16", False),
        # one token per stream
        _append("append_step", 64, 1, 120, 1000, 16, 64, "bf16"),
        # prompts of many requests, shared key heads
        _append("append_prompt", 12, 1000, 1000, 2500, 8, 128, "fp16"),
        # one layer of a few streams that reach max_model_len
        _evict("evict_layer", 4, 1, 700, 1000, 256, 34, 64, 16, 64),
        # every layer of eight streams: the conditioning rows and the last tokens stay
        _evict("evict_all_layers", 8, 30, 1500, 2011, 640, 34, 130, 16, 64),
        # a stream handed back to a 16-bit cache
        _read("read_streams", 5, 1500, 1500, 3001, 8, 128, 2, "bf16"),
    ]


def _attend(name, n, q, lo, hi, heads, kv, hd, dtype, weights):
    return {"name": name, "op": "attend", "n": n, "q": q, "lo": lo, "hi": hi, "heads": heads, "kv": kv, "hd": hd, "dtype": dtype, "weights": weights}


def _append(name, n, q, lo, hi, kv, hd, dtype):
    return {"name": name, "op": "append", "n": n, "q": q, "lo": lo, "hi": hi, "heads": kv, "kv": kv, "hd": hd, "dtype": dtype}


def _evict(name, n, layers, lo, hi, keep, sink, recent, kv, hd):
    return {"name": name, "op": "evict", "n": n, "layers": layers, "lo": lo, "hi": hi, "keep": keep, "sink": sink, "recent": recent,
            "kv": kv, "hd": hd, "dtype": "bf16"}


def _read(name, n, q, lo, hi, kv, hd, layers, dtype):
    return {"name": name, "op": "read", "n": n, "q": q, "lo": lo, "hi": hi, "kv": kv, "hd": hd, "layers": layers, "dtype": dtype}


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    largest = [work(c) for c in listed()]
    most_bytes = {op: max(w["bytes"] for w, c in zip(largest, listed()) if c["op"] == op) for op in ("attend", "append", "evict", "read")}
    most_flops = max(w["flops"] for w in largest)
    while True:
        op = rng.choice(("attend", "attend", "attend", "append", "evict", "read"))
        hd = rng.choice((64, 128))
        kv = rng.choice((1, 2, 3, 4, 8, 16))
        dtype = rng.choice(("bf16", "fp16"))
        if op == "attend":
            form = rng.choice(("decode", "decode", "draft", "prompt"))
            group = rng.choice((1, 1, 2, 3, 4, 5, 7, 8, 16))
            n = log(1, 128) if form == "decode" else log(1, 16)
            q = 1 if form == "decode" else rng.randint(2, 8) if form == "draft" else log(9, 4000)
            hi = max(q, log(1, 33000) if form != "prompt" else q + (0 if rng.random() < 0.5 else log(1, 2000)))
            c = _attend("", n, q, max(q, int(hi * rng.uniform(0.3, 1.0))), hi, kv * group, kv, hd, dtype, rng.random() < 0.5)
        elif op == "append":
            n = log(1, 64)
            q = 1 if rng.random() < 0.4 else log(2, 4000)
            hi = q + log(1, 4000) - 1
            c = _append("", n, q, max(q, int(hi * rng.uniform(0.3, 1.0))), hi, kv, hd, dtype)
        elif op == "evict":
            hi = log(40, 33000)
            keep = rng.randint(8, max(8, hi // 2))
            sink = rng.randint(0, keep // 4)
            c = _evict("", log(1, 16), log(1, 30), max(1, int(hi * rng.uniform(0.3, 1.0))), hi, keep, sink, rng.randint(0, keep // 2), kv, hd)
        else:
            q = log(1, 8000)
            hi = q + log(1, 2000) - 1
            c = _read("", log(1, 16), q, q, hi, kv, hd, log(1, 8), dtype)
        del c["name"]
        w = work(c)
        if w["bytes"] <= most_bytes[op] and w["flops"] <= most_flops and _room(c) < 6e9:
            return c


def _room(c):
    """Values of the largest tensor that the plain form makes, in bytes."""
    pages = _pages(c)
    keys = c["n"] * c.get("layers", 1) * c["kv"] * pages * PAGE * c["hd"] * 4
    return max(keys, c["n"] * c["heads"] * c["q"] * pages * PAGE * 4 if c["op"] == "attend" else 0)


def _lengths(c):
    """(rows, entries) of each sequence: spread over the case's range, the first one at its upper end."""
    ctx = [c["hi"] - int((c["hi"] - c["lo"]) * ((i * 0.6180339887498949) % 1.0)) for i in range(c["n"])]
    q = c.get("q", 0)
    rows = [q if q <= 16 else q - int((q // 2) * ((i * 0.7548776662466927) % 1.0)) for i in range(c["n"])]
    return [min(r, t) for r, t in zip(rows, ctx)], ctx


def _pages(c):
    return -(-c["hi"] // PAGE)


def _slab(hd):
    return PAGE * (hd + hd // 16)


def work(case):
    rows, ctx = _lengths(case)
    kv, hd, layers = case["kv"], case["hd"], case.get("layers", 1)
    entry = hd + hd // 16          # bytes of one (token, head): K and V codes, K and V scales
    if case["op"] == "attend":
        heads = case["heads"]
        seen = sum(r * (t - r) + r * (r + 1) // 2 for r, t in zip(rows, ctx))
        return {"bytes": sum(ctx) * kv * (entry + (8 if case["weights"] else 0)) + sum(rows) * heads * hd * 4, "flops": 4 * hd * heads * seen}
    if case["op"] in ("append", "read"):
        # append: the rows are read (16 bit), written as codes, read back as codes and handed out (16 bit)
        moved = layers * sum(rows) * kv
        return {"bytes": moved * (entry + 4 * hd) * (2 if case["op"] == "append" else 1), "flops": moved * 2 * hd}
    left = [min(t, case["keep"]) for t in ctx]
    width = _pages(case) * PAGE
    moved = layers * sum(left) * kv
    # weights of the source read, of the destination written; kept entries read and written, their indices written; then read back
    return {"bytes": layers * kv * (4 * sum(ctx) + 4 * width * len(ctx)) + moved * (2 * entry + 4) + moved * (entry + 4 * hd), "flops": moved * 2 * hd}


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    kv, hd, op, layers = case["kv"], case["hd"], case["op"], case.get("layers", 1)
    rows, ctx = _lengths(case)
    n, pages = case["n"], _pages(case)
    streams = 2 * n if op == "evict" else n                   # eviction: n sources and, behind them, n destinations
    dst_pages = -(-min(case.get("keep", 0), case["hi"]) // PAGE)
    used = n * pages + (n * dst_pages if op == "evict" else 0)
    num_pages = used + 3
    order = torch.randperm(num_pages, generator=g, device=dev)[:used].to(torch.int32)
    table = torch.zeros(streams, pages, dtype=torch.int32, device=dev)
    table[:n] = order[: n * pages].view(n, pages)
    if op == "evict":
        table[n:, :dst_pages] = order[n * pages:].view(n, dst_pages)

    # keys: unit channels with one in sixteen four times as large, and one token in sixteen along a direction that queries share
    gain = torch.ones(kv, hd, device=dev)
    gain[:, ::16] = 4.0
    lean = torch.randn(kv, 1, hd, generator=g, device=dev) * 0.6
    pool = torch.empty(layers, num_pages, kv, _slab(hd), dtype=torch.uint8, device=dev)
    at_once = max(1, (1 << 27) // (kv * PAGE * hd))
    for layer in range(layers):
        for a in range(0, num_pages, at_once):
            m = min(at_once, num_pages - a)
            k = torch.randn(m, kv, PAGE, hd, generator=g, device=dev) * gain[:, None]
            k += lean * (torch.rand(m, 1, PAGE, 1, generator=g, device=dev) < 1 / 16) * 1.5
            v = torch.randn(m, kv, PAGE, hd, generator=g, device=dev)
            pool[layer, a:a + m] = _to_slabs(*_quantise(k.to(torch.bfloat16)), *_quantise(v.to(torch.bfloat16)))
            del k, v
    s = {"case": dict(case), "pool": pool.view(layers, num_pages, kv * _slab(hd)), "table": table}

    if op in ("attend", "append", "read"):
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        s["streams"] = torch.randperm(n, generator=g, device=dev).to(torch.int32)
        s["seq_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device=dev)
        s["rows"], s["max_rows"], s["max_ctx"] = starts[-1], max(rows), max(ctx)
        owner = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(rows, device=dev))
        s["row_seq"], s["row_at"] = owner, torch.arange(starts[-1], device=dev) - s["seq_start"].long()[owner]
    if op in ("attend", "append"):
        heads = case["heads"]
        # the step's fused buffer q | k | v: the operators take views of it
        qkv = torch.randn(s["rows"], heads + 2 * kv, hd, generator=g, device=dev)
        qkv[:, heads:heads + kv] *= gain
        if op == "attend":
            qkv[:, :heads] = qkv[:, :heads] * (0.9 / math.sqrt(1 + 15 / 16)) + lean.repeat_interleave(heads // kv, 0)[:, 0]
        qkv = qkv.to(DTYPES[case["dtype"]])
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        s["scale"] = 1.0 / math.sqrt(hd)
    if case.get("weights"):
        s["weights"] = torch.rand(streams, kv, pages * PAGE, generator=g, device=dev)
    if op == "evict":
        # attention mass is heavy-tailed, and many entries were never looked at: those tie at zero
        w = torch.rand(layers, streams, kv, pages * PAGE, generator=g, device=dev)
        s["weights"] = torch.where(w < 0.15, torch.zeros_like(w), 1.0 / w.clamp_min(1e-6) - 1.0)
        s["src"] = torch.arange(n, dtype=torch.int32, device=dev)
        s["dst"] = torch.arange(n, 2 * n, dtype=torch.int32, device=dev)
        s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device=dev)
        left = [min(t, case["keep"]) for t in ctx]
        starts = [0]
        for r in left:
            starts.append(starts[-1] + r)
        s["left_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        s["left"] = torch.tensor(left, dtype=torch.int32, device=dev)
        s["rows"], s["max_rows"], s["max_ctx"] = starts[-1], max(left), max(ctx)
        owner = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(left, device=dev))
        s["row_seq"], s["row_at"] = owner, torch.arange(starts[-1], device=dev) - s["left_start"].long()[owner]
    return s


# ---------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _cache(s):
    """The cache object over the state's pool and block table, and the batch: made once, as a serving program keeps them."""
    if "cache" not in s:
        from chatterbox_vllm_amd.kv4_cache import KV4Cache
        c = s["case"]
        s["cache"] = KV4Cache(num_kv_heads=c["kv"], head_dim=c["hd"], pool=s["pool"], block_table=s["table"])
        if c["op"] == "evict":
            s["batch"] = s["cache"].batch(s["left_start"], s["dst"], s["left"], rows=s["rows"], max_rows=s["max_rows"], max_ctx=s["max_rows"])
        else:
            s["batch"] = s["cache"].batch(s["seq_start"], s["streams"], s["ctx"], rows=s["rows"], max_rows=s["max_rows"], max_ctx=s["max_ctx"])
    return s["cache"], s["batch"]


def _own_attend(s):
    cache, batch = _cache(s)
    out = cache.attend(s["q"], batch, scale=s["scale"], weights=s.get("weights"))
    return {"out": out, "weights": s.get("weights")}


def _own_append(s):
    cache, batch = _cache(s)
    cache.append(s["k"], s["v"], batch)
    k, v = cache.read(batch, dtype=DTYPES[s["case"]["dtype"]])
    return {"k": k, "v": v}


def _own_evict(s):
    cache, batch = _cache(s)
    c = s["case"]
    left, kept = cache.evict(s["src"], s["dst"], s["ctx"], keep=c["keep"], sink=c["sink"], recent=c["recent"], weights=s["weights"],
                             max_ctx=s["max_ctx"], n_layers=c["layers"])
    k, v = cache.read(batch, n_layers=c["layers"], dtype=DTYPES[c["dtype"]])
    return {"left": left, "kept": kept, "weights": s["weights"], "k": k, "v": v}


def _own_read(s):
    cache, batch = _cache(s)
    k, v = cache.read(batch, n_layers=s["case"]["layers"], dtype=DTYPES[s["case"]["dtype"]])
    return {"k": k, "v": v}


_OWN = {"attend": _own_attend, "append": _own_append, "evict": _own_evict, "read": _own_read}


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _quantise(x):
    """x [..., hd] -> codes [..., hd] and scale bytes [..., hd / 32] (uint8)."""
    x = x.float()
    blocks = x.view(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = blocks.abs().amax(-1)
    # the smallest power of two that leaves the block's largest value below 7, which still rounds to the largest code, 6
    b = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(2, 252)
    y = (blocks * torch.exp2((127 - b).float())[..., None]).reshape(x.shape)
    a = y.abs()
    r = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4)).clamp_max(7)
    return (r + torch.signbit(y) * 8).to(torch.uint8), b.to(torch.uint8)


def _value(codes, scales):
    """codes [..., hd] and scale bytes [..., hd / 32] -> fp32."""
    v = torch.tensor(LEVELS, dtype=torch.float32, device=codes.device)[codes.int()]
    step = torch.exp2(scales.float() - 127.0)
    return (v.view(*v.shape[:-1], -1, 32) * step[..., None]).view(v.shape)


def _fold(k, v):
    """K and V codes [..., 64, hd] -> bytes in slab order, [..., 32 hd] each.

    Both orders put side by side what one lane of a wave takes into a 16 x 16 x 32 matrix product in one 16-byte load: K, a
    quarter of the dims of one or two tokens; V, four dims of eight tokens."""
    hd, lead = k.shape[-1], k.shape[:-2]
    two = 128 // hd                                            # tokens whose quarter rows fill 16 bytes
    d = len(lead)
    k = k.reshape(*lead, 16, 4 // two, two, 4, hd // 8, 2)     # token 4 r + two i + j; dim quarter, byte, nibble
    k = k.permute(*range(d), d + 1, d + 3, d, d + 2, d + 4, d + 5)
    v = v.reshape(*lead, 4, 2, 8, hd // 64, 16, 2, 2)          # token 16 a + 8 b + c; dim 64 e + 4 r + 2 byte + nibble
    v = v.permute(*range(d), d + 3, d + 1, d, d + 4, d + 2, d + 5, d + 6)
    return tuple((x[..., 0] | x[..., 1] << 4).reshape(*lead, 32 * hd) for x in (k, v))


def _unfold(k, v, hd):
    """The inverse: bytes [..., 32 hd] each -> codes [..., 64, hd]."""
    lead = k.shape[:-1]
    two = 128 // hd
    d = len(lead)
    k = k.reshape(*lead, 4 // two, 4, 16, two, hd // 8)
    k = torch.stack([k & 15, k >> 4], -1).permute(*range(d), d + 2, d, d + 3, d + 1, d + 4, d + 5)
    v = v.reshape(*lead, hd // 64, 2, 4, 16, 8, 2)
    v = torch.stack([v & 15, v >> 4], -1).permute(*range(d), d + 2, d + 1, d + 4, d, d + 3, d + 5, d + 6)
    return k.reshape(*lead, PAGE, hd), v.reshape(*lead, PAGE, hd)


def _to_slabs(kc, ks, vc, vs):
    """Codes [..., 64, hd] and scales [..., 64, hd / 32] of whole pages -> slabs [..., bytes]."""
    k, v = _fold(kc, vc)
    return torch.cat([k, v, ks.transpose(-1, -2).flatten(-2), vs.transpose(-1, -2).flatten(-2)], -1)


def _from_slabs(slabs, hd):
    """slabs [..., bytes] -> K codes, K scales, V codes, V scales, a token a row."""
    half, nb = 32 * hd, hd // 32
    kc, vc = _unfold(slabs[..., :half], slabs[..., half:2 * half], hd)
    sc = slabs[..., 2 * half:].reshape(*slabs.shape[:-1], 2, nb, PAGE).transpose(-1, -2)
    return kc, sc[..., 0, :, :], vc, sc[..., 1, :, :]


def _stream_entries(s, layers, streams, pages):
    """Codes and scales of whole streams: four tensors [L, n, kv, 64 * pages, hd or hd / 32]."""
    c = s["case"]
    slabs = s["pool"].view(*s["pool"].shape[:2], c["kv"], -1)[:layers, s["table"][streams.long(), :pages].long()]   # [L, n, P, kv, slab]
    parts = _from_slabs(slabs, c["hd"])
    return tuple(p.transpose(2, 3).flatten(3, 4) for p in parts)


def _addresses(s, streams, slots):
    """Byte addresses, within one layer's pool, of row r's entry slots[r] in stream streams[row_seq[r]]: K codes and V codes
    [rows, kv, hd / 2] (two neighbouring dims a byte), K scales and V scales [rows, kv, hd / 32]."""
    kv, hd = s["case"]["kv"], s["case"]["hd"]
    page, t = s["table"][streams.long()[s["row_seq"]], slots // PAGE].long(), (slots % PAGE)[:, None, None]
    base = (page[:, None] * kv + torch.arange(kv, device=t.device))[..., None] * _slab(hd)
    byte, two = torch.arange(hd // 2, device=t.device), 128 // hd
    k_at = (t % 4 // two) * 1024 + ((byte // (hd // 8)) * 16 + t // 4) * 16 + (t % 4 % two) * 8 + byte % (hd // 8)
    v_at = 32 * hd + (byte // 32 * 2 + t // 8 % 2) * 1024 + ((t // 16) * 16 + byte % 32 // 2) * 16 + t % 8 * 2 + byte % 2
    s_at = 64 * hd + torch.arange(hd // 32, device=t.device) * PAGE + t
    return base + k_at, base + v_at, base + s_at, base + s_at + hd // 32 * PAGE


def _plain_read_rows(s, layers, streams, slots):
    """K and V of row r's entry slots[r] in stream streams[row_seq[r]]: [L, rows, kv, hd]."""
    out = DTYPES[s["case"]["dtype"]]
    flat, top = s["pool"][:layers].flatten(1), torch.finfo(out).max
    k, v, ks, vs = (flat[:, at] for at in _addresses(s, streams, slots))
    k, v = (_value(torch.stack([x & 15, x >> 4], -1).flatten(-2), b) for x, b in ((k, ks), (v, vs)))
    return k.clamp_(-top, top).to(out), v.clamp_(-top, top).to(out)


def _row_slots(s):
    n_rows = (s["seq_start"][1:] - s["seq_start"][:-1]).long()
    return (s["ctx"].long() - n_rows)[s["row_seq"]] + s["row_at"]


def _plain_attend(s):
    c = s["case"]
    kv, hd, heads = c["kv"], c["hd"], c["heads"]
    group, n, mq = heads // kv, c["n"], s["max_rows"]
    pages = -(-s["max_ctx"] // PAGE)
    kc, ks, vc, vs = _stream_entries(s, 1, s["streams"], pages)
    k, v = _value(kc[0], ks[0]), _value(vc[0], vs[0])                                   # [n, kv, T, hd]
    n_rows = (s["seq_start"][1:] - s["seq_start"][:-1]).long()
    j = torch.arange(mq, device=k.device)
    at = (s["seq_start"][:-1].long()[:, None] + j).clamp_max(s["rows"] - 1)
    q = s["q"][at].float().view(n, mq, kv, group, hd).transpose(1, 2).reshape(n, kv, mq * group, hd)
    seen = torch.where(j < n_rows[:, None], s["ctx"].long()[:, None] - n_rows[:, None] + j + 1, 0)      # [n, mq]
    t = torch.arange(pages * PAGE, device=k.device)
    hidden = (t >= seen[..., None]).repeat_interleave(group, 1)[:, None]                # [n, 1, mq * group, T]
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
    m = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    o = torch.matmul(p, v).view(n, kv, mq, group, hd).transpose(1, 2).reshape(n, mq, heads, hd)
    if "weights" in s:
        s["weights"][s["streams"].long(), :, : pages * PAGE] += p.sum(2)
    return {"out": o[s["row_seq"], s["row_at"]].to(DTYPES[c["dtype"]]), "weights": s.get("weights")}


def _plain_append(s):
    slots = _row_slots(s)
    k_at, v_at, ks_at, vs_at = _addresses(s, s["streams"], slots)
    (kc, ks), (vc, vs) = _quantise(s["k"]), _quantise(s["v"])
    flat = s["pool"][0].view(-1)
    flat[k_at], flat[v_at] = kc[..., ::2] | kc[..., 1::2] << 4, vc[..., ::2] | vc[..., 1::2] << 4
    flat[ks_at], flat[vs_at] = ks, vs
    k, v = _plain_read_rows(s, 1, s["streams"], slots)
    return {"k": k[0], "v": v[0]}


def _plain_read(s):
    k, v = _plain_read_rows(s, s["case"]["layers"], s["streams"], _row_slots(s))
    return {"k": k, "v": v}


def _plain_evict(s):
    c = s["case"]
    layers, kv, hd, n = c["layers"], c["kv"], c["hd"], c["n"]
    w = s["weights"][:, s["src"].long()]                                                # [L, n, kv, width]
    t = torch.arange(w.shape[-1], device=w.device)
    ctx = s["ctx"].long()[:, None]
    left = s["ctx"].clamp_max(c["keep"])
    # 0: stays in any case, 1: stays by its weight, 2: not an entry
    rank = torch.where(t >= ctx, 2, torch.where((t < c["sink"]) | (t >= ctx - c["recent"]) | (ctx <= c["keep"]), 0, 1))[None, :, None].expand(w.shape)
    order = torch.where(torch.isnan(w), -math.inf, w).argsort(dim=-1, descending=True, stable=True)
    order = order.gather(-1, rank.gather(-1, order).argsort(dim=-1, stable=True))[..., : c["keep"]]
    none = torch.arange(order.shape[-1], device=w.device) >= left.long()[:, None, None]
    order = order.masked_fill(none, w.shape[-1]).sort(-1).values
    kept = torch.where(order < w.shape[-1], order, -1).to(torch.int32)
    take = kept.long().clamp_min(0)
    pages = -(-min(c["keep"], c["hi"]) // PAGE)
    slots = torch.nn.functional.pad(take, (0, max(0, pages * PAGE - take.shape[-1])))[..., : pages * PAGE]
    parts = _stream_entries(s, layers, s["src"], _pages(c))
    parts = [x.gather(3, slots[..., None].expand(*slots.shape, x.shape[-1])).unflatten(3, (pages, PAGE)).transpose(2, 3) for x in parts]
    s["pool"].view(*s["pool"].shape[:2], kv, -1)[:, s["table"][s["dst"].long(), :pages].long()] = _to_slabs(*parts)
    moved = torch.where(kept < 0, 0.0, w.gather(-1, take))
    s["weights"][:, s["dst"].long()] = torch.nn.functional.pad(moved, (0, w.shape[-1] - c["keep"]))
    k, v = _plain_read_rows(s, layers, s["dst"], s["row_at"])
    return {"left": left, "kept": kept, "weights": s["weights"], "k": k, "v": v}


_PLAIN = {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict, "read": _plain_read}


# ---------------------------------------------------------------------------------------------------------------------
# What the outputs are by the operators' definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _entry(pool_layer, table_row, head, c, slots):
    """K and V [len(slots), hd] in 64 bits of entries `slots` of one stream and head: each code fetched by its own address."""
    kv, hd = c["kv"], c["hd"]
    t = slots % PAGE
    base = (table_row[slots // PAGE].long() * kv + head)[:, None] * (PAGE * hd + PAGE * hd // 16)
    d = torch.arange(hd, device=slots.device)[None]
    t = t[:, None]
    quarter = hd // 4
    if hd == 64:
        k_at = (t % 4 // 2) * 1024 + (d // quarter) * 256 + (t // 4) * 16 + (t % 2) * 8 + d % quarter // 2
    else:
        k_at = (t % 4) * 1024 + (d // quarter) * 256 + (t // 4) * 16 + d % quarter // 2
    v_at = 32 * hd + (d // 64) * 2048 + (t // 8 % 2) * 1024 + (t // 16) * 256 + (d % 64 // 4) * 16 + (t % 8) * 2 + d % 4 // 2
    flat = pool_layer.reshape(-1)
    codes = [(flat[base + at].long() >> (4 * (d % 2))) & 15 for at in (k_at, v_at)]
    scales = [flat[base + 64 * hd + which * 2 * hd + d // 32 * PAGE + t].double() for which in (0, 1)]
    out = []
    for code, b in zip(codes, scales):
        mag, e = (code & 1).double(), (code >> 1) & 3
        size = torch.where(e == 0, mag / 2, (1 + mag / 2) * torch.exp2(e.double() - 1))
        out.append(torch.where(code >= 8, -size, size) * torch.exp2(b - 127))
    return out


def _nearest(x):
    """What the cache holds of x [rows, kv, hd]: the nearest of the sixteen levels, ties to the even code, by comparison."""
    x = x.double()
    rows, kv, hd = x.shape
    blocks = x.view(rows, kv, hd // 32, 32)
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 7)).clamp(-125, 125)
    e = torch.where(top / torch.exp2(e) >= 7, e + 1, e)
    e = torch.where(top / torch.exp2(e - 1) < 7, e - 1, e).clamp(-125, 125)
    y = (blocks / torch.exp2(e)).abs()
    level = torch.tensor(LEVELS[:8], dtype=torch.float64, device=x.device)
    mid = (level[1:] + level[:-1]) / 2
    to_even = torch.arange(7, device=x.device) % 2 == 1        # halfway between an odd code and the even one above it: up
    code = ((y[..., None] > mid) | ((y[..., None] == mid) & to_even)).sum(-1)
    return (torch.copysign(level[code], blocks) * torch.exp2(e)).view(rows, kv, hd)


def exact(case, seed):
    s = prepare(case, seed)
    op, kv, n = case["op"], case["kv"], case["n"]
    dev = s["pool"].device
    if op == "append":
        return {"k": _nearest(s["k"]), "v": _nearest(s["v"])}
    rows, ctx = _lengths(case)
    if op == "read":
        ks, vs = [], []
        for layer in range(case["layers"]):
            for i in range(n):
                row = s["table"][int(s["streams"][i])]
                slots = torch.arange(ctx[i] - rows[i], ctx[i], device=dev)
                got = [_entry(s["pool"][layer], row, h, case, slots) for h in range(kv)]
                ks.append(torch.stack([k for k, _ in got], 1))
                vs.append(torch.stack([v for _, v in got], 1))
        shape = (case["layers"], sum(rows), kv, case["hd"])
        return {"k": torch.cat(ks).view(shape), "v": torch.cat(vs).view(shape)}
    if op == "attend":
        group = case["heads"] // kv
        out = torch.zeros(sum(rows), case["heads"], case["hd"], dtype=torch.float64, device=dev)
        weights = s["weights"].double() if case["weights"] else None
        first = 0
        for i in range(n):
            row, r, t = s["table"][int(s["streams"][i])], rows[i], ctx[i]
            slots = torch.arange(t, device=dev)
            bias = torch.zeros(r, t, dtype=torch.float64, device=dev).masked_fill(slots[None] > (t - r + torch.arange(r, device=dev))[:, None], -math.inf)
            for h in range(kv):
                k, v = _entry(s["pool"][0], row, h, case, slots)
                for head in range(h * group, (h + 1) * group):
                    p = torch.softmax(s["q"][first:first + r, head].double() @ k.t() / math.sqrt(case["hd"]) + bias, -1)
                    out[first:first + r, head] = p @ v
                    if weights is not None:
                        weights[int(s["streams"][i]), h, :t] += p.sum(0)
            first += r
        return {"out": out, "weights": weights}
    # evict: the kept set by sorting (weight, index) pairs on the host
    keep, width = case["keep"], s["weights"].shape[-1]
    layers = case["layers"]
    host = s["weights"].cpu().numpy()
    kept = torch.full((layers, n, kv, keep), -1, dtype=torch.int32)
    moved = torch.zeros(layers, n, kv, width, dtype=torch.float64)
    ks, vs = [], []
    for layer in range(layers):
        for i in range(n):
            got = []
            for h in range(kv):
                w, t = host[layer, i, h], ctx[i]
                if t <= keep:
                    stay = list(range(t))
                else:
                    a, b = case["sink"], t - case["recent"]
                    heavy = (-w[a:b]).argsort(kind="stable")[: keep - case["sink"] - case["recent"]] + a
                    stay = list(range(a)) + sorted(heavy.tolist()) + list(range(b, t))
                kept[layer, i, h, : len(stay)] = torch.tensor(stay, dtype=torch.int32)
                moved[layer, i, h, : len(stay)] = torch.from_numpy(w[stay]).double()
                got.append(_entry(s["pool"][layer], s["table"][i], h, case, torch.tensor(stay, device=dev)))
            ks.append(torch.stack([k for k, _ in got], 1))
            vs.append(torch.stack([v for _, v in got], 1))
    weights = s["weights"].double()
    weights[:, n:] = moved.to(dev)
    k, v = (torch.cat(x).view(layers, -1, kv, case["hd"]) for x in (ks, vs))
    return {"left": s["ctx"].clamp_max(keep), "kept": kept.to(dev), "weights": weights, "k": k, "v": v}
