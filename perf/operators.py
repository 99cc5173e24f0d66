"""The operators of serving from an 8-bit block cache, as measurable cases.

Four operators that run one after the other in each attention layer:

* ``norm_rope``: RMS norm of every query and key head and the rotation of its position;
* ``store``: new keys and values written to the block cache (8-bit codes, one scale for
  each block of tokens and head, per-channel bounds of the key codes), and the touched
  blocks read back;
* ``attend``: attention of one to a few query tokens a sequence over the whole cache;
* ``sparse``: the blocks with the largest bounds for the query chosen, and attention over
  these only.

``own = False`` computes them in elementary torch operations, ``own = True`` through
``unicache_b200``.  Sizes follow the repository's decode configurations (28 query and 4 KV
heads of 128 channels; 8192, 16384, 32768 and 131072 tokens; 16 to 64 sequences) and
generic ones around them.

Layouts: pool codes int8 [blocks, kv_heads, block, D], scales fp32 [blocks, kv_heads],
bounds int8 [blocks, kv_heads, D], pending rows [sequences, kv_heads, block, D] (the
unquantised rows of each sequence's incomplete block), table int32 [sequences, max_blocks],
lengths int32 [sequences] (after the write that a step makes).
"""

import math

import torch

own = False

TINY = 2.0 ** -120  # least scale: blocks of zeros have it


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a batch of 32
        {"name": "norm_rope_step", "op": "norm_rope", "tokens": 32, "q_heads": 28, "kv_heads": 4, "dim": 128,
         "rot": 128, "interleaved": False, "weights": True, "dtype": "bf16"},
        # a whole prompt of the benchmark's length
        {"name": "norm_rope_prompt", "op": "norm_rope", "tokens": 16384, "q_heads": 28, "kv_heads": 4, "dim": 128,
         "rot": 128, "interleaved": False, "weights": True, "dtype": "bf16"},
        # half of the channels rotated in adjacent pairs, no weights, an odd number of tokens
        {"name": "norm_rope_partial", "op": "norm_rope", "tokens": 4999, "q_heads": 16, "kv_heads": 2, "dim": 64,
         "rot": 32, "interleaved": True, "weights": False, "dtype": "f16"},
        # one token of each of 32 sequences appended in the middle of a block
        {"name": "store_step", "op": "store", "seqs": 32, "old": 1000, "new": 1, "kv_heads": 4, "dim": 128,
         "block": 64, "dtype": "bf16"},
        # four prompts of up to 16384 tokens written at once
        {"name": "store_prompts", "op": "store", "seqs": 4, "old": 0, "new": 16384, "kv_heads": 4, "dim": 128,
         "block": 64, "dtype": "bf16"},
        # a single short conversation: latency only
        {"name": "attend_one", "op": "attend", "seqs": 1, "tokens": 700, "ragged": False, "queries": 1,
         "q_heads": 28, "kv_heads": 4, "dim": 128, "block": 64, "dtype": "bf16"},
        # the benchmark's decode batch
        {"name": "attend_batch", "op": "attend", "seqs": 16, "tokens": 8192, "ragged": False, "queries": 1,
         "q_heads": 28, "kv_heads": 4, "dim": 128, "block": 64, "dtype": "bf16"},
        # a serving batch of unequal lengths (one token to the full length), smaller heads
        {"name": "attend_ragged", "op": "attend", "seqs": 48, "tokens": 16384, "ragged": True, "queries": 1,
         "q_heads": 32, "kv_heads": 8, "dim": 64, "block": 32, "dtype": "f16"},
        # four drafted tokens a sequence verified in one pass
        {"name": "attend_draft", "op": "attend", "seqs": 8, "tokens": 5003, "ragged": True, "queries": 4,
         "q_heads": 28, "kv_heads": 4, "dim": 128, "block": 64, "dtype": "bf16"},
        # the benchmark's long decode batch: over a gigabyte of cache
        {"name": "attend_long", "op": "attend", "seqs": 32, "tokens": 32768, "ragged": False, "queries": 1,
         "q_heads": 28, "kv_heads": 4, "dim": 128, "block": 64, "dtype": "bf16"},
        # one long document read through 32 of its blocks
        {"name": "sparse_one", "op": "sparse", "seqs": 1, "tokens": 30011, "ragged": False, "count": 32,
         "q_heads": 28, "kv_heads": 4, "dim": 128, "block": 64, "dtype": "bf16"},
        # eight sequences of 131072 tokens, 64 of 2048 blocks each
        {"name": "sparse_long", "op": "sparse", "seqs": 8, "tokens": 131072, "ragged": False, "count": 64,
         "q_heads": 28, "kv_heads": 4, "dim": 128, "block": 64, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "store", "attend", "sparse"])
    heads = rng.choice([(28, 4), (32, 8), (16, 2), (8, 8), (12, 4), (24, 3)])
    case = {"op": op, "q_heads": heads[0], "kv_heads": heads[1], "dim": rng.choice([64, 128, 128]),
            "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if op == "norm_rope":
        case["tokens"] = _log(rng, 1, 16384)
        case["rot"] = rng.choice([case["dim"], case["dim"], case["dim"] // 2])
        case["interleaved"] = rng.random() < 0.3
        case["weights"] = rng.random() < 0.8
        return case
    case["block"] = rng.choice([32, 64, 64, 128])
    if op == "store":
        del case["q_heads"]
        if rng.random() < 0.5:
            case.update(seqs=_log(rng, 1, 128), old=_log(rng, 1, 16384), new=1)
        else:
            case["seqs"] = _log(rng, 1, 8)
            case["old"] = case["block"] * rng.choice([0, 0, 3])
            case["new"] = _log(rng, 7, 65536 // case["seqs"])
        return case
    case["seqs"] = _log(rng, 1, 64)
    bytes_a_token = case["seqs"] * heads[1] * 2 * case["dim"]
    case["tokens"] = _log(rng, 1, max(2, min(131072, (1 << 29) // bytes_a_token)))
    case["ragged"] = rng.random() < 0.5
    if op == "attend":
        case["queries"] = rng.choice([1, 1, 1, 2, 5])
    else:
        case["count"] = _log(rng, 4, 128)
    return case


def _lengths(case):
    """Lengths of the sequences; ragged ones run from one token to the full length."""

    n, t = case["seqs"], case["tokens"]
    if not case["ragged"] or n == 1:
        return [t] * n
    return [1 + ((t - 1) * ((i * 7919) % n)) // (n - 1) for i in range(n)]


def _store_shape(case):
    """(tokens held before, tokens written) of each sequence."""

    n = case["seqs"]
    if case["new"] == 1:
        return [max(0, case["old"] - 37 * i) if i % 2 else case["old"] + 37 * i for i in range(n)], [1] * n
    return [case["old"]] * n, [max(1, case["new"] - i * (case["new"] // 5)) for i in range(n)]


def work(case):
    item = 2
    if case["op"] == "norm_rope":
        values = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * item * values + case["tokens"] * (case["rot"] * 4 + 8), "flops": 7 * values}
    d, b, h = case["dim"], case["block"], case["kv_heads"]
    if case["op"] == "store":
        old, new = _store_shape(case)
        written = sum(new)
        back = sum(o + n - o // b * b for o, n in zip(old, new))
        # rows in, codes out, codes in for the reading back, rows out
        return {"bytes": 2 * h * d * (item * written + written + back + item * back), "flops": 8 * h * d * written}
    lengths = _lengths(case)
    rows = case["seqs"] * case["q_heads"] * case.get("queries", 1)
    ends = rows * (2 * item * d + 4)
    if case["op"] == "attend":
        tokens = sum(lengths)
        return {"bytes": tokens * h * 2 * d + 8 * h * tokens // b + ends,
                "flops": 4 * d * case["q_heads"] * case["queries"] * tokens}
    blocks = [-(-t // b) for t in lengths]
    read = sum(min(case["count"] * b, t) for t in lengths)
    return {"bytes": sum(blocks) * h * (2 * d + 4) + read * h * 2 * d + ends,
            "flops": 4 * d * case["q_heads"] * (read + sum(blocks))}


# ---------------------------------------------------------------- inputs
def _dtype(case):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[case["dtype"]]


def _quantise(rows):
    """Codes, scales and bounds of [..., block, D] rows, as the cache holds them."""

    amax = rows.abs().amax(dim=(-2, -1))
    scale = (amax / torch.full_like(amax, 127.0)).clamp(min=TINY)
    codes = torch.round(rows * (1.0 / scale)[..., None, None]).clamp(-127, 127).to(torch.int8)
    return codes, scale


def _pool(case, gen, lengths, device):
    """A cache of full blocks with keys whose blocks differ in direction, its blocks in
    shuffled order, as they lie after some serving."""

    h, b, d, seqs = case["kv_heads"], case["block"], case["dim"], case["seqs"]
    width = max(1, -(-max(lengths) // b))
    blocks = seqs * width
    s = {"key_code": torch.empty(blocks, h, b, d, dtype=torch.int8, device=device),
         "value_code": torch.empty(blocks, h, b, d, dtype=torch.int8, device=device),
         "key_scale": torch.empty(blocks, h, device=device), "value_scale": torch.empty(blocks, h, device=device),
         "key_low": torch.empty(blocks, h, d, dtype=torch.int8, device=device),
         "key_high": torch.empty(blocks, h, d, dtype=torch.int8, device=device)}
    step = max(1, (1 << 26) // (h * b * d))
    for i in range(0, blocks, step):
        n = min(step, blocks - i)
        rows = torch.randn(n, h, b, d, generator=gen, device=device)
        rows += 0.7 * torch.randn(n, h, 1, d, generator=gen, device=device)
        codes, s["key_scale"][i:i + n] = _quantise(rows)
        s["key_code"][i:i + n] = codes
        s["key_low"][i:i + n], s["key_high"][i:i + n] = codes.amin(2), codes.amax(2)
        rows = torch.randn(n, h, b, d, generator=gen, device=device)
        s["value_code"][i:i + n], s["value_scale"][i:i + n] = _quantise(rows)
    s["block_table"] = torch.randperm(blocks, generator=gen, device=device).to(torch.int32).view(seqs, width)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    s["pending_key"] = torch.zeros(seqs, h, b, d, dtype=_dtype(case), device=device)
    s["pending_value"] = torch.zeros_like(s["pending_key"])
    return s


_TENSORS = ("key_code", "key_scale", "key_low", "key_high", "value_code", "value_scale", "pending_key",
            "pending_value", "block_table", "lengths")


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _dtype(case)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=device).to(dtype)

    if case["op"] == "norm_rope":
        t, hq, hk, d, rot = (case[k] for k in ("tokens", "q_heads", "kv_heads", "dim", "rot"))
        # query and key are views of one projection's output, as a decoder has them
        qkv = (2.5 * torch.randn(t, hq + 2 * hk, d, generator=gen, device=device)).to(dtype)
        inv_freq = 1.0 / (1e6 ** (torch.arange(rot // 2, device=device, dtype=torch.float64) / (rot // 2)))
        angle = torch.arange(32768, device=device, dtype=torch.float64)[:, None] * inv_freq
        weights = [(1.0 + 0.2 * torch.randn(d, generator=gen, device=device)).to(dtype) for _ in range(2)]
        start = 16384 if t <= 64 else 0
        if t <= 64:  # a decode step: every sequence has its own position
            positions = torch.randint(0, 32768, (t,), generator=gen, device=device, dtype=torch.int32)
        else:
            positions = torch.arange(start, start + t, device=device, dtype=torch.int32)
        return {"case": case, "query": qkv[:, :hq], "key": qkv[:, hq:hq + hk],
                "query_weight": weights[0] if case["weights"] else None,
                "key_weight": weights[1] if case["weights"] else None, "cos": angle.cos().float(),
                "sin": angle.sin().float(), "positions": positions, "eps": 1e-6}

    if case["op"] == "store":
        old, new = _store_shape(case)
        s = _pool(case, gen, [o + n for o, n in zip(old, new)], device)
        h, b, d, seqs = case["kv_heads"], case["block"], case["dim"], case["seqs"]
        held = torch.tensor([o % b for o in old], device=device)
        # rows held of the incomplete blocks, and these blocks as the cache holds them
        some = (torch.arange(b, device=device)[None] < held[:, None])[:, None, :, None]
        page = s["block_table"].gather(1, torch.tensor([[o // b] for o in old], device=device))[:, 0].long()
        for name in ("key", "value"):
            rows = randn(seqs, h, b, d) * some
            codes, scale = _quantise(rows.float())
            s["pending_" + name] = rows
            s[name + "_code"][page], s[name + "_scale"][page] = codes, scale
            if name == "key":
                s["key_low"][page] = torch.where(some, codes, 127).amin(2).to(torch.int8)
                s["key_high"][page] = torch.where(some, codes, -127).amax(2).to(torch.int8)
        s.update(case=case, key=randn(sum(new), h, d), value=randn(sum(new), h, d))
        back = [o + n - o // b * b for o, n in zip(old, new)]
        s["rows"] = sum(back)
        for name, counts in (("starts", new), ("back_starts", back)):
            s[name] = torch.tensor([sum(counts[:i]) for i in range(seqs + 1)], dtype=torch.int32, device=device)
        # blocks touched in all: the plan of a plain pass
        s["touched"] = sum(-(-n // b) for n in back)
    else:
        lengths = _lengths(case)
        s = _pool(case, gen, lengths, device)
        shape = (case["seqs"], case["queries"]) if case.get("queries", 1) > 1 else (case["seqs"],)
        s.update(case=case, query=randn(*shape, case["q_heads"], case["dim"]))
    if own:  # the cache object that a user's program keeps
        from unicache_b200 import Int8BlockCache

        s["cache"] = Int8BlockCache(**{k: s[k] for k in _TENSORS})
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    if op == "norm_rope":
        return _norm_rope(state)
    if op == "store":
        return _store(state)
    if op == "attend":
        return _attend(state, state["query"], None)
    blocks = _select(state)
    out, lse = _attend(state, state["query"], blocks)
    return blocks, out, lse


def _own(s, op):
    import unicache_b200 as ucb

    if op == "norm_rope":
        return ucb.head_norm_rope(s["query"], s["key"], s["query_weight"], s["key_weight"], s["cos"], s["sin"],
                                  s["positions"], eps=s["eps"], interleaved=s["case"]["interleaved"])
    cache = s["cache"]
    if op == "store":
        cache.write(s["key"], s["value"], starts=s["starts"])
        key, value = cache.read(s["rows"], starts=s["back_starts"])
        return key, value, cache.key_scale, cache.value_scale
    if op == "attend":
        return ucb.int8_block_decode(s["query"], cache)
    return ucb.sparse_int8_block_decode(s["query"], cache, count=s["case"]["count"], first=1, recent=2)


def _norm_rope(s):
    cos, sin = (s[k][s["positions"].long()][:, None] for k in ("cos", "sin"))
    rot, pairs = 2 * cos.shape[-1], s["case"]["interleaved"]

    def one(x, weight):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"])
        if weight is not None:
            y = y * weight.float()
        if pairs:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)

    return one(s["query"], s["query_weight"]), one(s["key"], s["key_weight"])


def _store(s):
    case, table = s["case"], s["block_table"].long()
    b, seqs, device = case["block"], case["seqs"], table.device
    length, starts = s["lengths"].long(), s["starts"].long()
    old = length - (starts[1:] - starts[:-1])
    first = old // b
    touched = (length - 1) // b - first + 1
    # every touched block of every sequence: its rows from the pending ones and the new ones
    seq = torch.repeat_interleave(torch.arange(seqs, device=device), touched, output_size=s["touched"])
    block = torch.arange(s["touched"], device=device) - (touched.cumsum(0) - touched)[seq] + first[seq]
    token = block[:, None] * b + torch.arange(b, device=device)
    is_new = (token >= old[seq][:, None])[:, None, :, None]
    held = (token < length[seq][:, None])[:, None, :, None]
    source = (starts[seq][:, None] + token - old[seq][:, None]).clamp(0, s["key"].shape[0] - 1)
    page, last = table[seq, block], (block == (length[seq] // b))
    for name in ("key", "value"):
        rows = torch.where(is_new, s[name][source].transpose(1, 2), s["pending_" + name][seq])
        rows = torch.where(held, rows, torch.zeros_like(rows))
        codes, scale = _quantise(rows.float())
        s[name + "_code"][page], s[name + "_scale"][page] = codes, scale
        if name == "key":
            s["key_low"][page] = torch.where(held, codes, 127).amin(2).to(torch.int8)
            s["key_high"][page] = torch.where(held, codes, -127).amax(2).to(torch.int8)
        # the incomplete block's rows stay pending; other blocks' go to a row that is dropped
        kept = torch.cat((s["pending_" + name], s["pending_" + name][:1]))
        kept[torch.where(last, seq, seqs)] = rows
        s["pending_" + name].copy_(kept[:seqs])
    # the touched blocks' rows read back
    back = s["back_starts"].long()
    seq = torch.repeat_interleave(torch.arange(seqs, device=device), back[1:] - back[:-1], output_size=s["rows"])
    token = torch.arange(s["rows"], device=device) - back[seq] + (length - (back[1:] - back[:-1]))[seq]
    page = table[seq, token // b]
    key, value = ((s[n + "_code"][page, :, token % b].float() * s[n + "_scale"][page][..., None]).to(s[n].dtype)
                  for n in ("key", "value"))
    return key, value, s["key_scale"], s["value_scale"]


def _select(s):
    case, q = s["case"], s["query"].float()
    seqs, h, count = case["seqs"], case["kv_heads"], case["count"]
    amax = q.abs().amax(-1, keepdim=True)
    q_scale = (amax / torch.full_like(amax, 127.0)).clamp(min=TINY)
    code = torch.round(q * (1.0 / q_scale)).clamp(-127, 127).view(seqs, h, -1, q.shape[-1])
    pages = s["block_table"].long()
    low, high = (s[k][pages].permute(0, 2, 3, 1).float() for k in ("key_low", "key_high"))
    bound = code.clamp(min=0) @ high + code.clamp(max=0) @ low  # whole numbers below 2^24: exact
    score = (bound * q_scale.view(seqs, h, -1, 1)).amax(2) * s["key_scale"][pages].transpose(1, 2)
    blocks = ((s["lengths"] + case["block"] - 1) // case["block"])[:, None, None]
    j = torch.arange(score.shape[-1], device=q.device)[None, None]
    score = torch.where((j < 1) | (j >= blocks - 2), math.inf, score)
    score = torch.where(j < blocks, score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :count]
    order = torch.where(order < blocks, order, score.shape[-1]).sort(-1).values
    order = torch.where(order < blocks, order, -1).to(torch.int32)
    return torch.nn.functional.pad(order, (0, count - order.shape[-1]), value=-1)


def _attend(s, query, blocks):
    case = s["case"]
    seqs, h, b, d, n = case["seqs"], case["kv_heads"], case["block"], case["dim"], case.get("queries", 1)
    q = query.float().view(seqs, n, h, -1, d).permute(0, 2, 1, 3, 4).reshape(seqs, h, -1, d)
    group = q.shape[2] // n
    table = s["block_table"].long()
    inside = torch.arange(b, device=q.device)
    if blocks is None:
        def gather(name):
            codes = s[name + "_code"][table].transpose(1, 2)
            return (codes.float() * s[name + "_scale"][table].transpose(1, 2)[..., None, None]).flatten(2, 3)
        token = torch.arange(table.shape[1] * b, device=q.device)[None, None]
    else:
        pages = table[:, None].expand(-1, h, -1).gather(2, blocks.long().clamp(min=0))
        head = torch.arange(h, device=q.device)[None, :, None]

        def gather(name):
            return (s[name + "_code"][pages, head].float() * s[name + "_scale"][pages, head][..., None, None]).flatten(2, 3)
        token = torch.where(blocks >= 0, blocks * b, 1 << 30)[..., None] + inside
        token = token.flatten(2)
    logits = (q @ gather("key").transpose(-1, -2)) / math.sqrt(d)
    limit = s["lengths"][:, None] - n + 1 + torch.arange(n, device=q.device)  # tokens that each query sees
    limit = limit.repeat_interleave(group, 1)[:, None, :, None]
    logits = torch.where(token[:, :, None] < limit, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(logits - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ gather("value")) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).view(seqs, h, n, group).transpose(1, 2).reshape(query.shape[:-1])
    out = out.view(seqs, h, n, group, d).transpose(1, 2).reshape(query.shape)
    return out.to(query.dtype), lse


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        return _exact_norm_rope(s)
    if case["op"] == "store":
        return _exact_store(s)
    if case["op"] == "attend":
        return _exact_attend(s, None)
    blocks = _exact_select(s)
    return (None, *_exact_attend(s, blocks))


def _exact_norm_rope(s):
    rot, device = 2 * s["cos"].shape[1], s["cos"].device
    channel = torch.arange(rot, device=device)
    if s["case"]["interleaved"]:
        partner, angle, sign = channel ^ 1, channel // 2, (channel % 2) * 2 - 1
    else:
        partner, angle, sign = (channel + rot // 2) % rot, channel % (rot // 2), (channel >= rot // 2) * 2 - 1
    at = s["positions"].long()
    cos, sin = (s[k].double()[at][:, angle][:, None] for k in ("cos", "sin"))
    outputs = []
    for x, w in ((s["query"], s["query_weight"]), (s["key"], s["key_weight"])):
        x = x.double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + s["eps"])
        y = y if w is None else y * w.double()
        z = y.clone()
        z[..., :rot] = y[..., :rot] * cos + sign * y[..., partner] * sin
        outputs.append(z)
    return tuple(outputs)


def _exact_store(s):
    b = s["case"]["block"]
    lengths, starts = s["lengths"].tolist(), s["starts"].tolist()
    outputs = []
    scales = {n: s[n + "_scale"].double() for n in ("key", "value")}
    for name in ("key", "value"):
        parts = []
        for i, length in enumerate(lengths):
            old = length - (starts[i + 1] - starts[i])
            pending = s["pending_" + name][i, :, :old % b].transpose(0, 1)
            rows = torch.cat((pending, s[name][starts[i]:starts[i + 1]])).double()
            size, blocks = rows.shape[0], -(-rows.shape[0] // b)
            rows = torch.cat((rows, rows.new_zeros(blocks * b - size, *rows.shape[1:]))).unflatten(0, (blocks, b))
            scale = (rows.abs().amax((1, 3)) / 127).clamp(min=TINY)
            codes = torch.round(rows / scale[:, None, :, None]).clamp(-127, 127)
            parts.append((codes * scale[:, None, :, None]).flatten(0, 1)[:size])
            pages = s["block_table"][i, old // b:old // b + blocks].long()
            scales[name][pages] = scale
        outputs.append(torch.cat(parts))
    return (*outputs, scales["key"], scales["value"])


def _exact_select(s):
    """Whole-number bounds and their products in the 32-bit steps that define the scores."""

    case = s["case"]
    b, count, h = case["block"], case["count"], case["kv_heads"]
    result = torch.full((case["seqs"], h, count), -1, dtype=torch.int64, device=s["query"].device)
    for i, length in enumerate(s["lengths"].tolist()):
        n = -(-length // b)
        pages = s["block_table"][i, :n].long()
        q = s["query"][i].float()
        top = q.abs().amax(1)
        scale = torch.maximum(top / torch.tensor([127.0], device=q.device), torch.tensor(TINY, device=q.device))
        code = torch.round(q * (1 / scale)[:, None]).clamp(-127, 127).double().view(h, -1, q.shape[1])
        for k in range(h):
            low, high = s["key_low"][pages, k].double(), s["key_high"][pages, k].double()
            most = torch.where(code[k] >= 0, code[k], 0.0) @ high.T + torch.where(code[k] < 0, code[k], 0.0) @ low.T
            score = (most.float() * scale.view(h, -1)[k][:, None]).amax(0) * s["key_scale"][pages, k]
            score = score.cpu().tolist()
            forced = {0} | set(range(max(0, n - 2), n))
            rest = sorted((j for j in range(n) if j not in forced), key=lambda j: (-score[j], j))
            kept = sorted(list(forced) + rest[:max(0, count - len(forced))])[:count]
            result[i, k, :len(kept)] = torch.tensor(kept, device=result.device)
    return result


def _exact_attend(s, blocks):
    case = s["case"]
    h, b, d, n = case["kv_heads"], case["block"], case["dim"], case.get("queries", 1)
    group = case["q_heads"] // h
    query = s["query"].double().view(case["seqs"], n, h, group, d)
    out, lse = torch.zeros_like(query), torch.full(query.shape[:-1], -math.inf, dtype=torch.float64, device=query.device)
    for i, length in enumerate(s["lengths"].tolist()):
        for k in range(h):
            chosen = torch.arange(-(-length // b), device=query.device) if blocks is None else blocks[i, k]
            chosen = chosen[chosen >= 0]
            pages = s["block_table"][i, chosen].long()
            key = (s["key_code"][pages, k].double() * s["key_scale"][pages, k].double()[:, None, None]).view(-1, d)
            value = (s["value_code"][pages, k].double() * s["value_scale"][pages, k].double()[:, None, None]).view(-1, d)
            token = (chosen[:, None] * b + torch.arange(b, device=query.device)).view(-1)
            for j in range(n):
                seen = token < length - n + 1 + j
                if not bool(seen.any()):
                    continue
                logits = query[i, j, k] @ key[seen].T / math.sqrt(d)
                lse[i, j, k] = torch.logsumexp(logits, -1)
                out[i, j, k] = torch.softmax(logits, -1) @ value[seen]
    return out.reshape(s["query"].shape), lse.reshape(s["query"].shape[:-1])
