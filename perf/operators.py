"""Performance cases of the attention operators: the per-head norms and position rotation of queries and keys,
writing a cache of 8-bit codes and reading it back, and attention over that cache.

The cache holds blocks of 64 tokens: codes of keys [blocks, heads, 64, dim] and of values
[blocks, heads, dim, 64] (int8 or e4m3), one fp32 scale for each block and head of either. A sequence's
blocks stand in its row of a table, anywhere in the pool. `own` False computes each operator in elementary
torch operations, `own` True calls `ishizuki_amd.attention`.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 64
DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LIMIT = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LEAST = 2.0 ** -126  # of a scale
EPS = 1e-6
BASE = 1e6


def _rotate(name, tokens, heads, kv_heads, dim, rot, dtype, interleaved=False, first=0):
    return {"name": name, "kind": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "dtype": dtype, "interleaved": interleaved, "first": first}


def _append(name, sequences, rows, length, heads, kv_heads, dim, rot, dtype, cache, ragged=False, fused=True):
    return {"name": name, "kind": "append", "sequences": sequences, "rows": rows, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rot": rot, "dtype": dtype, "cache": cache, "ragged": ragged,
            "fused": fused}


def _read(name, sequences, length, kv_heads, dim, dtype, cache, ragged=False):
    return {"name": name, "kind": "read", "sequences": sequences, "rows": 1, "length": length, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "cache": cache, "ragged": ragged}


def _attend(name, sequences, rows, length, heads, kv_heads, dim, dtype, cache, ragged=False, causal=True, window=0):
    return {"name": name, "kind": "attend", "sequences": sequences, "rows": rows, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "cache": cache, "ragged": ragged, "causal": causal,
            "window": window}


def listed():
    return [
        # one token's queries and keys between two projections of a decode step: launch and host latency
        _rotate("rotate_token", 1, 32, 8, 128, 128, "bf16"),
        # a prompt's, a quarter of each wide head rotated, far into a long context
        _rotate("rotate_prompt", 4096, 24, 4, 256, 64, "fp16", interleaved=True, first=1000003),
        # a decode step of a batch: norms and rotation, keys and values into partly filled blocks
        _append("append_step", 16, 1, 4096, 32, 8, 128, 128, "bf16", "int8", ragged=True),
        # a prompt's keys and values, as they are, into fresh blocks
        _append("append_prompt", 1, 8192, 8192, 32, 8, 128, 128, "fp16", "e4m3", fused=False),
        # a short conversation read back for a draft model's own layout
        _read("read_short", 1, 200, 4, 64, "fp16", "e4m3"),
        # long contexts read back to be kept or moved
        _read("read_long", 2, 32768, 8, 128, "bf16", "int8", ragged=True),
        # one token of one conversation
        _attend("decode_short", 1, 1, 777, 32, 8, 128, "bf16", "int8"),
        # a decode step of a batch with long contexts, one slot of it idle
        _attend("decode_batch", 16, 1, 32768, 32, 8, 128, "bf16", "int8", ragged=True),
        # eight drafted tokens of each sequence verified, wide heads
        _attend("verify_wide", 4, 8, 8191, 32, 4, 256, "fp16", "e4m3"),
        # a whole prompt
        _attend("prompt", 1, 8192, 8192, 32, 8, 128, "bf16", "int8"),
        # pieces of three prompts behind what their caches hold, each token seeing 4096 back
        _attend("pieces_window", 3, 1500, 12000, 16, 2, 64, "bf16", "e4m3", ragged=True, window=4096),
        # a decoder's tokens over an encoder's states: no order between the two
        _attend("cross", 2, 333, 1500, 16, 16, 64, "fp16", "int8", causal=False),
    ]


def _spread(rng, low, high):
    """A whole number of low..high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "read", "attend", "attend"])
    most = [work(c) for c in listed() if c["kind"] == kind]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        dim = rng.choice([64, 128, 256])
        rot = rng.choice([dim, dim // 2, dim // 4])
        kv = rng.choice([1, 2, 3, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        dtype = rng.choice(["bf16", "fp16"])
        cache = rng.choice(["int8", "e4m3"])
        ragged = rng.random() < 0.5
        sequences = _spread(rng, 1, 32)
        length = _spread(rng, 1, 65536)
        rows = rng.choice([1, 1, _spread(rng, 2, 16), _spread(rng, 1, 8192)])
        rows = min(rows, length)
        if kind == "rotate":
            case = _rotate("", _spread(rng, 1, 8192), heads, kv, dim, rot, dtype, rng.random() < 0.3,
                           rng.choice([0, 131071, 1000003]))
        elif kind == "append":
            case = _append("", sequences, rows, length, heads, kv, dim, rot, dtype, cache, ragged, rng.random() < 0.6)
        elif kind == "read":
            case = _read("", sequences, length, kv, dim, dtype, cache, ragged)
        else:
            causal = rng.random() < 0.8
            window = _spread(rng, 1, length) if causal and rng.random() < 0.3 else 0
            case = _attend("", sequences, rows, length, heads, kv, dim, dtype, cache, ragged, causal, window)
            if sequences * rows * heads * length > 1 << 31:  # the plain form's scores
                continue
        if kind != "rotate" and sequences * length * kv * dim > 1 << 30:  # the pool
            continue
        w = work(case)
        if all(w[k] <= most[k] for k in most):
            del case["name"]
            return case


def _rows_lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence. A ragged batch goes down to half the rows and
    three eighths of the length, and from four sequences on its last slot is idle."""
    n, count, length = case["sequences"], case["rows"], case["length"]
    if not case["ragged"]:
        return [(count, length)] * n
    out = []
    for s in range(n):
        rows = max(1, count - s * count // (2 * n))
        out.append((rows, max(rows, length - s * 5 * length // (8 * n) - (s * 37) % 64)))
    if n >= 4:
        out[-1] = (0, 0)
    return out


def work(case):
    item = DTYPE[case["dtype"]].itemsize
    dim, kv = case["dim"], case["kv_heads"]
    if case["kind"] == "rotate":
        values = case["tokens"] * (case["heads"] + kv) * dim
        return {"bytes": 2 * values * item + 4 * case["tokens"] + 8 * dim + 4 * case["rot"], "flops": 10 * values}
    seqs = _rows_lengths(case)
    tokens = sum(n for n, _ in seqs)
    blocks = sum(-(-length // BLOCK) for _, length in seqs)
    if case["kind"] == "append":
        values = 2 * tokens * kv * dim
        back = 2 * sum(min(length, n + BLOCK) for n, length in seqs) * kv * dim
        q = 2 * tokens * case["heads"] * dim * item if case["fused"] else 0
        return {"bytes": values * (item + 1) + q + back * item, "flops": 4 * values + 10 * q / item + back}
    if case["kind"] == "read":
        held = 2 * sum(length for _, length in seqs) * kv * dim
        return {"bytes": held * (1 + item) + 8 * blocks * kv, "flops": held}
    window, pairs, seen = case["window"], 0, 0
    for n, length in seqs:
        if not case["causal"]:
            pairs, seen = pairs + n * length, seen + length
            continue
        first = length - n
        for i in range(n):
            pairs += min(first + i + 1, window) if window else first + i + 1
        seen += min(length, n - 1 + window) if window and n else length if n else 0
    return {"bytes": 2 * seen * kv * dim + 8 * -(-seen // BLOCK) * kv + 2 * tokens * case["heads"] * dim * item,
            "flops": 4 * pairs * case["heads"] * dim}


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _channels(g, heads, dim):
    """Sizes of a head's channels: some are several times the others, as keys' are."""
    return 1.0 + 4.0 * (torch.rand(heads, dim, generator=g, device=DEV) < 0.04).float()


def _pool(g, case):
    """A pool's codes and scales as writing whole blocks leaves them."""
    kv, dim, code = case["kv_heads"], case["dim"], CODE[case["cache"]]
    blocks = sum(-(-length // BLOCK) for _, length in _rows_lengths(case)) + 3
    held = {"k": torch.empty((blocks, kv, BLOCK, dim), dtype=code, device=DEV),
            "v": torch.empty((blocks, kv, dim, BLOCK), dtype=code, device=DEV),
            "k_scale": torch.empty((blocks, kv), device=DEV), "v_scale": torch.empty((blocks, kv), device=DEV)}
    part = max(1, (1 << 26) // (kv * BLOCK * dim))
    wide = _channels(g, kv, dim)
    for name, by in (("k", wide[:, None, :]), ("v", 1.0)):
        for b in range(0, blocks, part):
            x = torch.randn(held[name][b:b + part].shape, generator=g, device=DEV) * by
            scale = x.abs().amax((-1, -2)) / LIMIT[code]
            x = x / scale[..., None, None]
            held[name][b:b + part] = (torch.round(x) if code is torch.int8 else x).to(code)
            held[name + "_scale"][b:b + part] = scale
    return held


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype, dim, kv = DTYPE[case["dtype"]], case["dim"], case["kv_heads"]
    state = {"case": case}
    if case["kind"] == "rotate" or case["kind"] == "append":
        rot, heads = case["rot"], case["heads"]
        inv = BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
        state["inv_freq"] = inv.to(DEV)
        # the same rates in turns a position, as 64-bit fractions
        state["turns"] = torch.tensor([int(f / (2 * math.pi) * 2.0 ** 64) for f in inv.tolist()], device=DEV)
        state["q_weight"] = 1.0 + 0.2 * _normal(g, dim)
        state["k_weight"] = 1.0 + 0.2 * _normal(g, dim)
        tokens = case["tokens"] if case["kind"] == "rotate" else sum(n for n, _ in _rows_lengths(case))
        # the projection's output holds q, k and v side by side
        qkv = _normal(g, tokens, heads + 2 * kv, dim)
        qkv[:, heads:heads + kv] *= _channels(g, kv, dim)
        qkv = qkv.to(dtype)
        state["q"], state["k"], state["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    if case["kind"] == "rotate":
        state["positions"] = torch.arange(case["first"], case["first"] + case["tokens"], dtype=torch.int32, device=DEV)
        return state
    seqs = _rows_lengths(case)
    state["cache"] = tuple(_pool(g, case).values())
    widths = [-(-length // BLOCK) for _, length in seqs]
    order = torch.randperm(state["cache"][0].shape[0], generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(seqs), max(widths) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, w in enumerate(widths):
        table[s, :w] = order[at:at + w]
        at += w
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    state["table"] = table
    state["lengths"] = torch.tensor([length for _, length in seqs], dtype=torch.int32, device=DEV)
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    state["max_rows"], state["max_length"] = max(n for n, _ in seqs), max(length for _, length in seqs)
    if case["kind"] == "append":
        for scale in state["cache"][2:]:  # what some blocks hold so far is smaller than what comes
            scale *= torch.where(torch.rand(scale.shape, generator=g, device=DEV) < 0.3, 0.3, 1.0)
        state["tail"] = min(state["max_length"], state["max_rows"] + BLOCK)
        state["positions"] = torch.cat([torch.arange(length - n, length, dtype=torch.int32, device=DEV) for n, length in seqs])
    if case["kind"] == "attend":
        state["q"] = _normal(g, starts[-1], case["heads"], dim).to(dtype)
    return state


def _plain_norm_rope(x, weight, s):
    """x [tokens, heads, dim] in 32 bits; the angles in 64."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    rot = 2 * s["inv_freq"].numel()
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if s["case"].get("interleaved"):
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _rows(s):
    """(sequence, place in it) of each row of the call, for any number of rows in a sequence."""
    row = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(s["starts"].long(), row, right=True) - 1
    return seq, row - s["starts"].long()[seq]


def _plain_quantize(x, codes, scales, block, slot, lead, transposed):
    """The new tokens' x [tokens, heads, dim] into their blocks: a block that starts with them gets the scale of
    their largest value, one that goes on (among `lead`, each sequence's first) keeps its own unless that is too
    small, and then grows it by the least power of two."""
    limit = LIMIT[codes.dtype]
    blocks, heads = scales.shape
    most = x.abs().amax(-1)
    amax = torch.zeros((blocks, heads), device=DEV).scatter_reduce(0, block[:, None].expand(-1, heads), most, "amax")
    first = torch.full((blocks,), BLOCK, device=DEV).scatter_reduce(0, block, slot, "amin")
    held = limit * scales
    (ma, ea), (mb, eb) = torch.frexp(amax), torch.frexp(held)
    grow = torch.where(amax <= held, 0, ea - eb + (ma > mb).int())
    fresh = (amax / limit).clamp(min=LEAST)
    scale = torch.where((first == 0)[:, None], fresh, torch.ldexp(scales, grow))
    scale = torch.where((first < BLOCK)[:, None], scale, scales)
    grow = torch.where(((first > 0) & (first < BLOCK))[:, None], grow, 0)
    bits = codes.view(torch.int8)
    old = torch.ldexp(bits[lead].view(codes.dtype).float(), -grow[lead][..., None, None])
    old = torch.round(old) if codes.dtype is torch.int8 else old
    bits[lead] = old.to(codes.dtype).view(torch.int8)
    scales.copy_(scale)
    new = (x / scale[block][..., None]).clamp(-limit, limit)
    new = (torch.round(new) if codes.dtype is torch.int8 else new).to(codes.dtype)
    if transposed:
        bits[block, :, :, slot] = new.view(torch.int8)
    else:
        bits[block, :, slot] = new.view(torch.int8)


def _plain_read(s, codes, scales, tail, transposed, dtype):
    """The last `tail` tokens of each sequence, zeros where it has fewer."""
    at = s["lengths"].long()[:, None] - tail + torch.arange(tail, device=DEV)
    there = at >= 0
    at = at.clamp(min=0)
    block = s["table"].long().gather(1, at // BLOCK).clamp(min=0)
    slot = at % BLOCK
    bits = codes.view(torch.int8)
    x = bits[block, :, :, slot] if transposed else bits[block, :, slot]
    x = x.view(codes.dtype).float() * scales[block][..., None]
    return torch.where(there[..., None, None], x, 0.0).to(dtype)


def _plain_attend(s):
    case = s["case"]
    k, v, k_scale, v_scale = s["cache"]
    kv, dim, group = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    most, table = s["max_rows"], s["table"].long().clamp(min=0)
    n = table.shape[1] * BLOCK
    keys = (k.view(torch.int8)[table].view(k.dtype).float() * k_scale[table][..., None, None]).permute(0, 2, 4, 1, 3).reshape(-1, kv, dim, n)
    seq, place = _rows(s)
    row = (s["starts"][:-1, None].long() + torch.arange(most, device=DEV)).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].reshape(-1, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(-1, kv, most * group, dim)
    scores = torch.matmul(q, keys) * dim ** -0.5
    del keys
    token = torch.arange(n, device=DEV)
    length, rows = s["lengths"].long()[:, None, None], (s["starts"][1:] - s["starts"][:-1]).long()[:, None, None]
    seen = token < length
    if case["causal"]:
        position = length - rows + torch.arange(most, device=DEV)[:, None]
        seen = seen & (token <= position)
        if case["window"]:
            seen = seen & (token > position - case["window"])
    seen = seen.expand(-1, most, -1)[:, None, :, None].expand(-1, 1, -1, group, -1).reshape(-1, 1, most * group, n)
    scores.masked_fill_(~seen, -math.inf)
    peak = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(peak).exp_()
    total = p.sum(-1, keepdim=True)
    values = (v.view(torch.int8)[table].view(v.dtype).float() * v_scale[table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(-1, kv, n, dim)
    out = torch.matmul(p, values) / torch.where(total == 0, 1.0, total)
    out = out.reshape(-1, kv, most, group, dim)[seq, :, place]
    return out.reshape(-1, case["heads"], dim).to(s["q"].dtype)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        from ishizuki_amd import attention
        if kind == "rotate":
            return attention.norm_rope(state["q"], state["k"], state["positions"], state["turns"], state["q_weight"],
                                       state["k_weight"], eps=EPS, interleaved=case["interleaved"])
        cache = attention.Cache(*state["cache"])
        batch = attention.Batch(state["table"], state["lengths"], state["starts"], state["max_rows"], state["max_length"])
        if kind == "read":
            return attention.read(cache, batch, dtype=DTYPE[case["dtype"]])
        if kind == "attend":
            return attention.attend(state["q"], cache, batch, causal=case["causal"], window=case["window"])
        if case["fused"]:
            q = attention.append(state["k"], state["v"], cache, batch, q=state["q"], positions=state["positions"],
                                 turns=state["turns"], q_weight=state["q_weight"], k_weight=state["k_weight"], eps=EPS)
        else:
            q = None
            attention.append(state["k"], state["v"], cache, batch)
        k, v = attention.read(cache, batch, tail=state["tail"], dtype=DTYPE[case["dtype"]])
        return {"q": q, "k": k, "v": v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    if kind == "rotate":
        dtype = state["q"].dtype
        return (_plain_norm_rope(state["q"], state["q_weight"], state).to(dtype),
                _plain_norm_rope(state["k"], state["k_weight"], state).to(dtype))
    if kind == "attend":
        return _plain_attend(state)
    k, v, k_scale, v_scale = state["cache"]
    dtype = DTYPE[case["dtype"]]
    if kind == "read":
        return (_plain_read(state, k, k_scale, state["max_length"], False, dtype),
                _plain_read(state, v, v_scale, state["max_length"], True, dtype))
    q, new_k = None, state["k"].float()
    if case["fused"]:
        q = _plain_norm_rope(state["q"], state["q_weight"], state).to(dtype)
        new_k = _plain_norm_rope(state["k"], state["k_weight"], state)
    seq, place = _rows(state)
    at = (state["lengths"] - state["starts"][1:] + state["starts"][:-1]).long()[seq] + place
    block, slot = state["table"].long()[seq, at // BLOCK], at % BLOCK
    lead = block[state["starts"][:-1].long().clamp(max=block.shape[0] - 1)]
    _plain_quantize(new_k, k, k_scale, block, slot, lead, False)
    _plain_quantize(state["v"].float(), v, v_scale, block, slot, lead, True)
    return {"q": q, "k": _plain_read(state, k, k_scale, state["tail"], False, dtype),
            "v": _plain_read(state, v, v_scale, state["tail"], True, dtype), "k_scale": k_scale, "v_scale": v_scale}


def _exact_turned(x, weight, case, positions):
    """Per-head norm and rotation as complex products in 64 bits."""
    x = x.double()
    x = weight.double() * x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    half = case["rot"] // 2
    rate = torch.tensor([BASE ** (-2.0 * i / case["rot"]) for i in range(half)], dtype=torch.float64, device=DEV)
    wheel = torch.polar(torch.ones_like(rate), positions.double()[:, None, None] * rate)
    pairs = torch.complex(x[..., 0:2 * half:2].contiguous(), x[..., 1:2 * half:2].contiguous()) if case.get("interleaved") else \
        torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous())
    pairs = pairs * wheel
    out = x.clone()
    if case.get("interleaved"):
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = pairs.real, pairs.imag
    else:
        out[..., :half], out[..., half:2 * half] = pairs.real, pairs.imag
    return out


def _exact_store(values, scales, new, table, first, limit, round_):
    """One sequence's new [tokens, heads, dim] into values [blocks, heads, 64, dim] (codes as 64-bit numbers), block
    by block; returns the blocks touched."""
    touched, at = [], 0
    while at < new.shape[0]:
        b, slot = int(table[(first + at) // BLOCK]), (first + at) % BLOCK
        count = min(BLOCK - slot, new.shape[0] - at)
        x = new[at:at + count].transpose(0, 1)
        most = x.abs().amax((1, 2))
        if slot == 0:
            scales[b] = (most / limit).clamp(min=LEAST)
        else:
            over = torch.log2(most / (limit * scales[b])).ceil().clamp(min=0)
            scales[b] *= 2 ** over
            values[b] = round_(values[b] / 2 ** over[:, None, None])
        values[b, :, slot:slot + count] = round_((x / scales[b][:, None, None]).clamp(-limit, limit))
        touched.append(b)
        at += count
    return touched


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rotate":
        return (_exact_turned(state["q"], state["q_weight"], case, state["positions"]),
                _exact_turned(state["k"], state["k_weight"], case, state["positions"]))
    k, v, k_scale, v_scale = state["cache"]
    table, seqs = state["table"].tolist(), _rows_lengths(case)
    starts = state["starts"].tolist()
    kv, dim = case["kv_heads"], case["dim"]

    def tokens(codes, scales, s, first, last, transposed):
        """Tokens first..last of sequence s and their values in 64 bits, [heads, tokens, dim]."""
        blocks = table[s][first // BLOCK:-(-last // BLOCK)]
        x = codes.view(torch.int8)[blocks].view(codes.dtype).double() * scales[blocks].double()[..., None, None]
        x = x.transpose(-1, -2) if transposed else x
        x = x.transpose(0, 1).reshape(kv, -1, dim)
        return x[:, first % BLOCK:first % BLOCK + last - first]

    if case["kind"] == "attend":
        group, window, out = case["heads"] // kv, case["window"], []
        for s, (n, length) in enumerate(seqs):
            if not n:
                continue
            keys, values = (tokens(*a, s, 0, length, t) for a, t in (((k, k_scale), False), ((v, v_scale), True)))
            position = torch.arange(length - n, length, device=DEV)
            token = torch.arange(length, device=DEV)
            q = state["q"][starts[s]:starts[s] + n].double().reshape(n, kv, group, dim)
            got = torch.empty((n, kv, group, dim), dtype=torch.float64, device=DEV)
            for h in range(kv):
                for j in range(group):
                    score = q[:, h, j] @ keys[h].T / math.sqrt(dim)
                    if case["causal"]:
                        hidden = token > position[:, None]
                        if window:
                            hidden |= token <= position[:, None] - window
                        score = score.masked_fill(hidden, -math.inf)
                    got[:, h, j] = torch.softmax(score, -1) @ values[h]
            out.append(got.reshape(n, case["heads"], dim))
        return torch.cat(out)
    back = state["max_length"]
    if case["kind"] == "append":
        back = state["tail"]
        new_k = state["k"].double()
        if case["fused"]:
            new_k = _exact_turned(state["k"], state["k_weight"], case, state["positions"])
        if k.dtype is torch.int8:
            round_ = torch.round
        else:
            def round_(x):  # three bits after the leading one, and steps of 2^-9 below 2^-6
                step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
                return torch.round(x / step) * step
        for codes, scales, new, transposed in ((k, k_scale, new_k, False), (v, v_scale, state["v"].double(), True)):
            held, wide = codes.double(), scales.double()
            held = held.transpose(-1, -2).contiguous() if transposed else held
            for s, (n, length) in enumerate(seqs):
                _exact_store(held, wide, new[starts[s]:starts[s] + n], table[s], length - n, LIMIT[codes.dtype], round_)
            if transposed:
                v, v_scale = held.transpose(-1, -2), wide
            else:
                k, k_scale = held, wide
    got = []
    for codes, scales, transposed in ((k, k_scale, False), (v, v_scale, True)):
        x = torch.zeros((len(seqs), back, kv, dim), dtype=torch.float64, device=DEV)
        for s, (_, length) in enumerate(seqs):
            first = max(0, length - back)
            blocks = table[s][first // BLOCK:-(-length // BLOCK)]
            y = codes[blocks].double() if codes.dtype is torch.float64 else codes.view(torch.int8)[blocks].view(codes.dtype).double()
            y = y * scales[blocks].double()[..., None, None]
            y = (y.transpose(-1, -2) if transposed else y).transpose(1, 2).reshape(-1, kv, dim)
            y = y[first - first // BLOCK * BLOCK:]
            x[s, back - (length - first):] = y[:length - first]
        got.append(x)
    if case["kind"] == "read":
        return tuple(got)
    q = _exact_turned(state["q"], state["q_weight"], case, state["positions"]) if case["fused"] else None
    return {"q": q, "k": got[0], "v": got[1], "k_scale": k_scale, "v_scale": v_scale}
