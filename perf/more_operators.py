"""The operators of a serving step around the 8-bit block cache, as measurable cases.

Five operators that a batch needs beside the cache's write and attention:

* ``verify``: drafted tokens accepted or rejected against the target's distribution from given
  random numbers, the next token drawn from what remains, the rejected tokens taken off the lengths;
* ``admit``: blocks of finished sequences given back to the pool and blocks for new prompts taken;
* ``fork``: sequences continued in several others: complete blocks shared, the incomplete one
  copied in every layer;
* ``compact``: the live blocks of a fragmented pool moved to its front, in every layer;
* ``axes``: RMS norm of every query and key head and the rotation by positions of several axes
  (time, height and width of image and video tokens).

``own = False`` computes them in elementary torch operations, ``own = True`` through
``unicache_b200``.  Sizes follow the repository's decoder (28 layers, 28 query and 4 KV heads of 128
channels, a vocabulary of 151936, blocks of 64 tokens) and generic ones around them.

Layouts: logits [sequences, drafts + 1, vocabulary]; pool codes int8 [layers, blocks, kv_heads, block, D], scales
fp32 [layers, blocks, kv_heads], bounds int8 [layers, blocks, kv_heads, D], pending rows [layers, sequences,
kv_heads, block, D]; table int32 [sequences, max_blocks] (-1: none), lengths int32 [sequences],
references int32 [blocks] (how many table entries name a block).
"""

import math

import torch

own = False


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one conversation with four drafted tokens: latency only
        {"name": "verify_one", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 32000, "logits": "bf16", "probs": "f32",
         "temperature": "one", "ragged": False},
        # a serving batch with a draft model, its requests' temperatures mixed, some of them greedy
        {"name": "verify_batch", "op": "verify", "seqs": 32, "drafts": 4, "vocab": 151936, "logits": "bf16",
         "probs": "f32", "temperature": "mixed", "ragged": False},
        # drafts looked up in the prompt (no draft distribution), of unequal numbers; an odd vocabulary
        {"name": "verify_lookup", "op": "verify", "seqs": 48, "drafts": 7, "vocab": 50257, "logits": "f16", "probs": "none",
         "temperature": "mixed", "ragged": True},
        # the largest batch, logits kept in fp32
        {"name": "verify_large", "op": "verify", "seqs": 64, "drafts": 7, "vocab": 151936, "logits": "f32", "probs": "bf16",
         "temperature": "one", "ragged": False},
        # a quarter of 32 sequences ends, and as many prompts come in
        {"name": "admit_batch", "op": "admit", "seqs": 32, "tokens": 16384, "groups": 4, "block": 64, "spare": 0.1},
        # the same for a node's whole pool: 2048 sequences, small blocks
        {"name": "admit_many", "op": "admit", "seqs": 2048, "tokens": 2011, "groups": 8, "block": 32, "spare": 0.25},
        # one prompt continued in eight samples, two layers
        {"name": "fork_samples", "op": "fork", "seqs": 8, "parents": 1, "tokens": 1003, "layers": 2, "kv_heads": 4,
         "dim": 128, "block": 64, "dtype": "bf16"},
        # eight prompts in eight samples each, the whole decoder
        {"name": "fork_batch", "op": "fork", "seqs": 64, "parents": 8, "tokens": 4090, "layers": 28, "kv_heads": 4,
         "dim": 128, "block": 64, "dtype": "bf16"},
        # a small pool of one layer
        {"name": "compact_layer", "op": "compact", "seqs": 12, "groups": 3, "tokens": 1500, "layers": 1, "kv_heads": 8,
         "dim": 64, "block": 32, "dtype": "f16", "spare": 0.2},
        # a quarter of the sequences has ended: the whole decoder's pool
        {"name": "compact_pool", "op": "compact", "seqs": 48, "groups": 4, "tokens": 2048, "layers": 28, "kv_heads": 4,
         "dim": 128, "block": 64, "dtype": "bf16", "spare": 0.1},
        # frames of a video of the benchmark's prompt length, time, height and width in sections
        {"name": "axes_video", "op": "axes", "tokens": 16384, "q_heads": 28, "kv_heads": 4, "dim": 128, "rot": 128,
         "axes": 3, "alternating": False, "interleaved": False, "weights": True, "dtype": "bf16"},
        # one image, height and width by turns, half of the channels in adjacent pairs; an odd number of tokens
        {"name": "axes_image", "op": "axes", "tokens": 4999, "q_heads": 16, "kv_heads": 2, "dim": 64, "rot": 32,
         "axes": 2, "alternating": True, "interleaved": True, "weights": False, "dtype": "f16"},
    ]


def _log(rng, low, high):
    high = max(low, high)
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["verify", "verify", "admit", "fork", "compact", "axes"])
    if op == "verify":
        vocab, drafts = _log(rng, 1000, 200000), rng.choice([0, 1, 2, 3, 4, 5, 7, 8, 15])
        return {"op": op, "seqs": _log(rng, 1, max(1, min(256, 75_000_000 // (vocab * (drafts + 1))))), "drafts": drafts,
                "vocab": vocab, "logits": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "probs": rng.choice(["f32", "f32", "bf16", "none"]), "temperature": rng.choice(["one", "mixed"]),
                "ragged": rng.random() < 0.3}
    if op == "axes":
        heads = rng.choice([(28, 4), (32, 8), (16, 2), (8, 8), (12, 4), (24, 3)])
        dim = rng.choice([64, 128, 128])
        return {"op": op, "tokens": _log(rng, 1, 16384), "q_heads": heads[0], "kv_heads": heads[1], "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2]), "axes": rng.choice([2, 3, 3, 4]),
                "alternating": rng.random() < 0.4, "interleaved": rng.random() < 0.3, "weights": rng.random() < 0.8,
                "dtype": rng.choice(["bf16", "bf16", "f16"])}
    case = {"op": op, "block": rng.choice([16, 32, 64, 64, 128])}
    if op == "admit":
        seqs = _log(rng, 2, 1024)
        case.update(seqs=seqs, tokens=_log(rng, 17, min(32768, 4_000_000 // seqs)), groups=rng.choice([2, 3, 8]) if seqs > 8 else 2,
                    spare=rng.choice([0.0, 0.1, 0.5]))
        return case
    heads, dim = rng.choice([(4, 128), (8, 64), (8, 128), (2, 128)])
    layers = rng.choice([1, 2, 7, 28])
    seqs = _log(rng, 4, 64)
    # the pool's codes take 1.5 GB at most
    most = (3 << 29) // (seqs * layers * heads * 2 * dim)
    case.update(seqs=seqs, tokens=_log(rng, 17, min(4096, max(18, most - 2 * case["block"]))), layers=layers, kv_heads=heads, dim=dim,
                dtype=rng.choice(["bf16", "bf16", "f16"]))
    if op == "fork":
        case["parents"] = _log(rng, 1, max(1, seqs // 3))
    else:
        case.update(groups=rng.choice([2, 3, 4]), spare=rng.choice([0.0, 0.1, 0.5]))
    return case


def _lengths(case):
    """Unequal lengths up to the case's tokens, none below a quarter of them."""

    n, t = case["seqs"], case["tokens"]
    return [max(1, t - (3 * t // 4) * ((i * 7919) % n) // n) for i in range(n)]


def _width(case):
    return -(-case["tokens"] // case["block"]) + 1


def _counts(case):
    n = case["drafts"]
    return [(i * 5) % (n + 1) if case["ragged"] else n for i in range(case["seqs"])]


def _sizes():
    return {"bf16": 2, "f16": 2, "f32": 4, "none": 0}


def work(case):
    op = case["op"]
    if op == "verify":
        rows = sum(n + 1 for n in _counts(case))
        item, q_item = _sizes()[case["logits"]], _sizes()[case["probs"]]
        # every row of logits, and of the draft's distributions the one that the new token is drawn from
        drawn = sum(n > 0 for n in _counts(case))
        return {"bytes": case["vocab"] * (rows * item + drawn * q_item) + 32 * rows, "flops": 4 * rows * case["vocab"]}
    if op == "axes":
        values = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 4 * values + case["tokens"] * case["rot"] * 4 + 4 * case["tokens"] * case["axes"], "flops": 7 * values}
    b, lengths = case["block"], _lengths(case)
    if op == "admit":
        # the references read, and the entries of the sequences that end and come written
        turned = sum(-(-t // b) for t in lengths) // case["groups"]
        return {"bytes": 4 * _blocks(case) + 24 * turned + 12 * case["seqs"], "flops": 0}
    head = case["layers"] * case["kv_heads"]
    if op == "fork":
        total = 4 * _blocks(case)
        for i, parent in enumerate(_pairs(case)[0]):
            held = lengths[parent] % b
            # codes of the rows held, the rows themselves, scales and bounds, read and written; the shared entries
            total += 2 * head * (held * case["dim"] * (2 + 4) + (8 + 2 * case["dim"]) * (held > 0)) + 12 * (lengths[parent] // b)
        return {"bytes": total, "flops": 0}
    moved = sum(-(-t // b) for t in lengths) // case["groups"]
    return {"bytes": 2 * moved * head * (2 * b * case["dim"] + 8 + 2 * case["dim"]) + 4 * _blocks(case) + 8 * case["seqs"] * _width(case),
            "flops": 0}


# ---------------------------------------------------------------- inputs
def _dtype(name):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _pairs(case):
    """Parents and children of a fork: the first sequences are the parents, all others continue one of them."""

    children = list(range(case["parents"], case["seqs"]))
    return [i % case["parents"] for i in children], children


def _blocks(case):
    """Blocks of the pool: those of all sequences, and some spare ones."""

    held = sum(-(-t // case["block"]) for t in _lengths(case))
    return held + case["seqs"] + int(case.get("spare", 0.0) * held)


def _held(case, gen, device):
    """A pool whose sequences' blocks lie anywhere in it, as after some serving."""

    lengths, width, blocks = _lengths(case), _width(case), _blocks(case)
    lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
    used = (lengths + case["block"] - 1) // case["block"]
    inside = torch.arange(width, device=device)[None] < used[:, None]
    place = torch.randperm(blocks, generator=gen, device=device).to(torch.int32)
    rank = (inside.flatten().cumsum(0) - 1).clamp(min=0).view_as(inside)
    table = torch.where(inside, place[rank], -1).to(torch.int32)
    references = torch.zeros(blocks, dtype=torch.int32, device=device)
    references[place[:int(used.sum())].long()] = 1
    return {"block_table": table, "lengths": lengths, "references": references}


def _layers(case, gen, device):
    """Contents of all layers' caches; a layer is a slice of each."""

    n, h, b, d = case["layers"], case["kv_heads"], case["block"], case["dim"]
    blocks = _blocks(case)
    s = {}
    for name in ("key", "value"):
        s[name + "_code"] = torch.randint(-127, 128, (n, blocks, h, b, d), generator=gen, device=device, dtype=torch.int8)
        s[name + "_scale"] = 0.01 + 0.02 * torch.rand(n, blocks, h, generator=gen, device=device)
        s["pending_" + name] = torch.randn(n, case["seqs"], h, b, d, generator=gen, device=device, dtype=_dtype(case["dtype"]))
    s["key_low"] = torch.randint(-127, 0, (n, blocks, h, d), generator=gen, device=device, dtype=torch.int8)
    s["key_high"] = torch.randint(0, 128, (n, blocks, h, d), generator=gen, device=device, dtype=torch.int8)
    return s


_STATE = ("key_code", "value_code", "key_scale", "value_scale", "key_low", "key_high", "pending_key", "pending_value")


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, gen, device)
    if case["op"] == "axes":
        return _prepare_axes(case, gen, device)
    s = {"case": case, "turn": 0, **_held(case, gen, device)}
    if case["op"] == "fork":
        s["parents"], s["children"] = (torch.tensor(x, dtype=torch.int32, device=device) for x in _pairs(case))
    else:
        # which sequences end in each pass, and the tokens of the prompts that take their places
        groups = [list(range(g, case["seqs"], case["groups"])) for g in range(case["groups"])]
        s["ends"] = [torch.tensor(g, dtype=torch.int32, device=device) for g in groups]
        s["prompts"] = []
        for g in s["ends"]:
            tokens = torch.zeros_like(s["lengths"])
            tokens[g.long()] = s["lengths"][g.long()]
            s["prompts"].append(tokens)
        # the plan of a plain pass: no more blocks move than there are places behind the live ones
        used = [-(-t // case["block"]) for t in _lengths(case)]
        stay = [sum(used) - sum(used[i] for i in g) for g in groups]
        s["moves"] = max(min(n, _blocks(case) - n) for n in stay)
    if case["op"] != "admit":
        s.update(_layers(case, gen, device))
    if own:  # the pool and the layers' caches that a user's program keeps
        from unicache_b200 import BlockPool, Int8BlockCache

        s["pool"] = BlockPool(block_table=s["block_table"], lengths=s["lengths"], references=s["references"],
                              block_size=case["block"])
        if case["op"] != "admit":
            s["pool"].attach([Int8BlockCache(block_table=s["block_table"], lengths=s["lengths"], **{k: s[k][i] for k in _STATE})
                              for i in range(case["layers"])])
    return s


def _prepare_verify(case, gen, device):
    seqs, n, vocab = case["seqs"], case["drafts"], case["vocab"]

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=device)

    # logits with a few likely tokens over a long tail, as a language model gives them
    z = 2.0 * torch.randn(seqs, n + 1, vocab, generator=gen, device=device)
    likely = torch.randint(0, vocab, (seqs, n + 1, 16), generator=gen, device=device)
    z.scatter_add_(2, likely, 4.0 + 9.0 * rand(seqs, n + 1, 16))
    s = {"case": case, "logits": z.to(_dtype(case["logits"])), "uniforms": rand(seqs, n + 1), "draft_probs": None,
         "temperature": None}
    heat = torch.ones(seqs, device=device)
    if case["temperature"] == "mixed":  # a quarter greedy, the others from 0.5 to 1.5
        heat = torch.where(torch.arange(seqs, device=device) % 4 == 3, 0.0, 0.5 + rand(seqs))
        s["temperature"] = heat
    scale = (1.0 / torch.where(heat > 0, heat, 0.05))[:, None, None]
    if case["probs"] == "none":
        # drafts that were looked up: often the target's likely token, sometimes any
        best = z[:, :n].argmax(-1)
        s["drafts"] = torch.where(rand(seqs, n) < 0.75, best, torch.randint(0, vocab, (seqs, n), generator=gen, device=device))
    else:
        z = z[:, :n]
        z += 0.7 * torch.randn(seqs, n, vocab, generator=gen, device=device)
        probs = torch.softmax(z * scale, -1).to(_dtype(case["probs"]))
        s["draft_probs"] = probs
        noise = -torch.log(rand(seqs, n, vocab).clamp(min=1e-30))
        s["drafts"] = (probs.float() / noise).argmax(-1)
    s["drafts"] = s["drafts"].to(torch.int32)
    s["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=device)
    # far from zero, as every pass takes rejected tokens off
    s["lengths"] = torch.randint(1 << 24, 1 << 25, (seqs,), generator=gen, device=device, dtype=torch.int32)
    return s


def _prepare_axes(case, gen, device):
    t, hq, hk, d, rot, axes = (case[k] for k in ("tokens", "q_heads", "kv_heads", "dim", "rot", "axes"))
    dtype = _dtype(case["dtype"])
    # query and key are views of one projection's output, as a decoder has them
    qkv = (2.5 * torch.randn(t, hq + 2 * hk, d, generator=gen, device=device)).to(dtype)
    inv_freq = 1.0 / (1e6 ** (torch.arange(rot // 2, device=device, dtype=torch.float64) / (rot // 2)))
    angle = torch.arange(32768, device=device, dtype=torch.float64)[:, None] * inv_freq
    weights = [(1.0 + 0.2 * torch.randn(d, generator=gen, device=device)).to(dtype) for _ in range(2)]
    # rows of a picture of some width, frame after frame, behind some text
    wide, high = 40, 25
    start = int(torch.randint(0, 1000, (1,), generator=gen, device=device))
    i = torch.arange(t, device=device)
    grid = torch.stack((i // (wide * high), i // wide % high, i % wide, i % 7))
    positions = start + (grid[:3] if axes == 3 else grid[1:3] if axes == 2 else grid)
    half = rot // 2
    if case["alternating"]:  # pair i turns by axis i mod axes
        axis = [k % axes for k in range(half)]
    else:  # sections: the first axis has the smallest
        first = half // (axes + 1) // 4 * 4
        rest = (half - first) // (axes - 1)
        sections = [first] + [rest] * (axes - 2) + [half - first - rest * (axes - 2)]
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    return {"case": case, "query": qkv[:, :hq], "key": qkv[:, hq:hq + hk],
            "query_weight": weights[0] if case["weights"] else None,
            "key_weight": weights[1] if case["weights"] else None, "cos": angle.cos().float(), "sin": angle.sin().float(),
            "positions": positions.to(torch.int32).contiguous(), "axis": tuple(axis),
            "axis_of_pair": torch.tensor(axis, device=device), "eps": 1e-6}


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    g = state.get("turn", 0)
    if op in ("admit", "compact"):  # every pass ends another group of sequences
        state["turn"] = (g + 1) % state["case"]["groups"]
    if own:
        return _own(state, op, g)
    if op == "verify":
        return _verify(state)
    if op == "axes":
        return _axes(state)
    if op == "fork":
        _fork(state)
        return _state(state)
    _release(state, state["ends"][g].long())
    live = _compact(state) if op == "compact" else None
    _advance(state, state["prompts"][g])
    return live, _state(state)


def _state(s):
    """Table, lengths and references, and the contents that were moved: whole codes, and rows as they are."""

    return [s[k] for k in ("block_table", "lengths", "references", *_STATE) if k in s]


def _own(s, op, g):
    import unicache_b200 as ucb

    if op == "verify":
        return (*ucb.verify_drafts(s["logits"], s["drafts"], s["uniforms"], draft_probs=s["draft_probs"],
                                   temperature=s["temperature"], counts=s["counts"], lengths=s["lengths"]), s["lengths"])
    if op == "axes":
        return ucb.head_norm_rope(s["query"], s["key"], s["query_weight"], s["key_weight"], s["cos"], s["sin"],
                                  s["positions"], eps=s["eps"], interleaved=s["case"]["interleaved"], axes=s["axis"])
    pool = s["pool"]
    if op == "fork":
        pool.fork(s["parents"], s["children"])
        return _state(s)
    pool.release(s["ends"][g])
    live = pool.compact() if op == "compact" else None
    pool.advance(s["prompts"][g])
    return live, _state(s)


def _verify(s):
    """In 64 bits: the tokens depend on sums over the vocabulary next to borders."""

    logits, drafts, counts, u = s["logits"].double(), s["drafts"].long(), s["counts"].long(), s["uniforms"].double()
    seqs, rows, vocab = logits.shape
    n, device = rows - 1, logits.device
    heat = torch.ones(seqs, device=device) if s["temperature"] is None else s["temperature"]
    greedy = heat <= 0
    top = logits.amax(-1, keepdim=True)
    index = torch.arange(vocab, device=device)
    best = torch.where(logits == top, index, vocab).amin(-1)
    x = (logits - top) / torch.where(greedy, 1.0, heat).double()[:, None, None]
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    seq, j = torch.arange(seqs, device=device), torch.arange(rows, device=device)
    p_draft = (e[:, :n].gather(2, drafts[..., None]) / total[:, :n])[..., 0]
    if s["draft_probs"] is None:
        q_draft = torch.ones_like(p_draft)
    else:
        q_draft = s["draft_probs"].gather(2, drafts[..., None])[..., 0].double()
    ok = torch.where(greedy[:, None], drafts == best[:, :n], u[:, :n] * q_draft < p_draft)
    ok &= j[None, :n] < counts[:, None]
    accepted = ok.long().cumprod(1).sum(1)
    # the next token: from what the draft's distribution leaves of the target's
    p = e[seq, accepted] / total[seq, accepted]
    rejected = accepted < counts
    if n == 0:
        q = torch.zeros_like(p)
    elif s["draft_probs"] is None:
        q = (index[None] == drafts[seq, accepted.clamp(max=n - 1)][:, None]).double()
    else:
        q = s["draft_probs"][seq, accepted.clamp(max=n - 1)].double()
    left = (p - torch.where(rejected[:, None], q, 0.0)).clamp(min=0)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, p)
    running = left.cumsum(-1)
    token = (running <= u[:, n:] * running[:, -1:]).sum(-1).clamp(max=vocab - 1)
    token = torch.where(greedy, best[seq, accepted], token)
    out = torch.cat((drafts, drafts.new_zeros(seqs, 1)), 1)
    out = torch.where(j < accepted[:, None], out, torch.where(j == accepted[:, None], token[:, None], -1))
    logprob = (x.gather(2, out.clamp(min=0)[..., None]) - torch.log(total))[..., 0]
    logprob = torch.where(j <= accepted[:, None], logprob, 0.0)
    s["lengths"] -= (counts - accepted).int()
    return out.int(), accepted.int(), logprob.float(), s["lengths"]


def _free_order(references):
    """Free blocks in ascending order (then the others), and how many they are."""

    taken = references > 0
    return torch.sort(taken.int(), stable=True).indices, (~taken).sum()


def _release(s, ends):
    table, references = s["block_table"], s["references"]
    rows = table[ends]
    held = rows >= 0
    references.index_add_(0, rows.clamp(min=0).flatten().long(), -held.flatten().int())
    table[ends] = -1
    s["lengths"][ends] = 0


def _advance(s, tokens):
    table, references, b = s["block_table"], s["references"], s["case"]["block"]
    old = s["lengths"].clone()
    s["lengths"] += tokens
    j = torch.arange(table.shape[1], device=table.device)[None]
    want = (j >= (old // b)[:, None]) & (j < ((s["lengths"] + b - 1) // b)[:, None]) & (table < 0)
    rank = (want.flatten().cumsum(0) - 1).view_as(want)
    order, free = _free_order(references)
    given = want & (rank < free)
    table.copy_(torch.where(given, order[rank.clamp(0, references.numel() - 1)].int(), table))
    references.index_add_(0, table.clamp(min=0).flatten().long(), given.flatten().int())


def _fork(s):
    table, references, lengths, b = s["block_table"], s["references"], s["lengths"], s["case"]["block"]
    parents, children = s["parents"].long(), s["children"].long()
    _release(s, children)
    held = lengths[parents]
    rows = table[parents]
    j = torch.arange(table.shape[1], device=table.device)[None]
    last, inside = (held // b)[:, None], (held % b)[:, None]
    shared = j < last
    references.index_add_(0, rows.clamp(min=0).flatten().long(), (shared & (rows >= 0)).flatten().int())
    copied = (inside > 0)[:, 0]
    order, free = _free_order(references)
    # a pair without an incomplete block copies its first block to itself
    to = torch.where(copied, order[(copied.cumsum(0) - 1).clamp(min=0)], rows[:, 0].clamp(min=0).long())
    table[children] = torch.where(shared, rows, torch.where((j == last) & copied[:, None], to[:, None].int(), -1)).int()
    references.index_add_(0, to, copied.int())
    lengths[children] = held
    # the incomplete blocks, in every layer
    source = rows.gather(1, last.clamp(max=table.shape[1] - 1).long())[:, 0].clamp(min=0).long()
    source = torch.where(copied, source, to)
    some = (torch.arange(b, device=table.device)[None] < inside)[None, :, None, :, None]
    for name in ("key", "value"):
        codes, pending = s[name + "_code"], s["pending_" + name]
        codes[:, to] = torch.where(some, codes[:, source], codes[:, to])
        kept = some.clone()
        if name == "key":  # and the record of whose rows they are
            kept[..., -1:, :] = copied[None, :, None, None, None]
        pending[:, children] = torch.where(kept, pending[:, parents], pending[:, children])
        s[name + "_scale"][:, to] = s[name + "_scale"][:, source]
    for name in ("key_low", "key_high"):
        s[name][:, to] = s[name][:, source]


def _compact(s):
    table, references = s["block_table"], s["references"]
    n = references.numel()
    live = references > 0
    count = live.sum()
    i = torch.arange(n, device=table.device)
    hole, mover = ~live & (i < count), live & (i >= count)
    holes = torch.sort((~hole).int(), stable=True).indices[:s["moves"]]
    movers = torch.sort((~mover).int(), stable=True).indices[:s["moves"]]
    # what is left of the plan copies the last pair again (with nothing to move, a block to itself)
    k = torch.minimum(torch.arange(holes.numel(), device=table.device), (mover.sum() - 1).clamp(min=0))
    to, source = holes[k], movers[k]
    place = i.clone()
    place[source] = to
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()].int(), table))
    references[to] = references[source]
    references[i >= count] = 0
    for name in _STATE[:6]:
        s[name][:, to] = s[name][:, source]
    return count.int().view(1)


def _axes(s):
    case = s["case"]
    at = s["positions"].long()[s["axis_of_pair"]].t()  # [tokens, pairs]
    cos, sin = (s[k].gather(0, at)[:, None] for k in ("cos", "sin"))
    rot, pairs = case["rot"], case["interleaved"]

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


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    if case["op"] == "verify":
        return _exact_verify(prepare(case, seed))
    if case["op"] == "axes":
        return _exact_axes(prepare(case, seed))
    return None  # blocks are moved, nothing is computed


def _exact_verify(s):
    """Sequence by sequence, a draft after the other; the tokens are whole numbers, the log-probabilities are not."""

    seqs, rows, vocab = s["logits"].shape
    heats = [1.0] * seqs if s["temperature"] is None else s["temperature"].tolist()
    counts, drafts, u = s["counts"].tolist(), s["drafts"].tolist(), s["uniforms"].double().tolist()
    result = torch.zeros(seqs, rows, dtype=torch.float64)
    for i in range(seqs):
        heat = heats[i] if heats[i] > 0 else 1.0
        j = 0
        while True:
            logs = torch.log_softmax(s["logits"][i, j].double() / heat, -1)
            if j == counts[i]:
                left = logs.exp()
                break
            x = drafts[i][j]
            if heats[i] <= 0:
                stays = int((logs == logs.max()).nonzero()[0]) == x
            else:
                q = 1.0 if s["draft_probs"] is None else float(s["draft_probs"][i, j, x])
                stays = u[i][j] * q < math.exp(float(logs[x]))
            if stays:
                result[i, j] = float(logs[x])
                j += 1
                continue
            if s["draft_probs"] is None:
                left = logs.exp()
                left[x] = 0.0
            else:
                left = torch.relu(logs.exp() - s["draft_probs"][i, j].double())
            break
        if heats[i] <= 0:
            token = int((logs == logs.max()).nonzero()[0])
        else:
            if not float(left.sum()) > 0:
                left = logs.exp()
            running = torch.cumsum(left, 0)
            token = int(torch.searchsorted(running, u[i][rows - 1] * running[-1:], right=True).clamp(max=vocab - 1))
        result[i, j] = float(logs[token])
    return None, None, result, None


def _exact_axes(s):
    rot, device = s["case"]["rot"], s["cos"].device
    channel = torch.arange(rot, device=device)
    if s["case"]["interleaved"]:
        partner, pair, sign = channel ^ 1, channel // 2, (channel % 2) * 2 - 1
    else:
        partner, pair, sign = (channel + rot // 2) % rot, channel % (rot // 2), (channel >= rot // 2) * 2 - 1
    at = torch.stack([s["positions"][a] for a in s["axis"]], 1).long()
    cos, sin = (s[k].double()[at[:, pair], pair[None]][:, None] for k in ("cos", "sin"))
    outputs = []
    for x, w in ((s["query"], s["query_weight"]), (s["key"], s["key_weight"])):
        x = x.double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + s["eps"])
        y = y if w is None else y * w.double()
        z = y.clone()
        z[..., :rot] = y[..., :rot] * cos + sign * y[..., partner] * sin
        outputs.append(z)
    return tuple(outputs)
