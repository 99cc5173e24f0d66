"""Draft verification against its definition in 64 bits: tokens and counts exactly, log-probabilities within the roundings
of an fp32 sum."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle.verify import verify
from unicache_b200 import kernels, verify_drafts

from .gpu_util import host, need_gpu

pytestmark = pytest.mark.gpu

BAD = 2  # the device error bit
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(seqs, n, vocab, *, dtype=torch.bfloat16, probs=torch.float32, heat=None, seed=0, near=0.7):
    """Logits with likely tokens over a tail, draft distributions near the target's, drafts drawn from them."""

    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    z = 2 * torch.randn(seqs, n + 1, vocab, generator=gen, device="cuda")
    z.scatter_add_(2, torch.randint(0, vocab, (seqs, n + 1, 12), generator=gen, device="cuda"), 3 + 8 * rand(seqs, n + 1, 12))
    t = torch.ones(seqs, device="cuda") if heat is None else heat
    t = torch.where(t > 0, t, 0.05)[:, None, None]
    q = torch.softmax((z[:, :n] + near * torch.randn(seqs, n, vocab, generator=gen, device="cuda")) / t, -1)
    drafts = (q / -torch.log(rand(seqs, n, vocab).clamp(min=1e-30))).argmax(-1)
    return z.to(dtype), drafts, rand(seqs, n + 1), None if probs is None else q.to(probs)


def check(logits, drafts, uniforms, draft_probs=None, temperature=None, counts=None, *, unclear=0, **more):
    """All sequences against the oracle.  A test nearer to its border than the fp32 sum's error, or a draw nearer than fp64's, may
    fall either way: `unclear` such sequences at most."""

    seqs, rows, vocab = logits.shape
    lengths = torch.arange(100, 100 + seqs, device="cuda", dtype=torch.int32)
    before = [x.clone() for x in (logits, drafts, uniforms)]
    kernels.device_status()
    tokens, accepted, logprobs = verify_drafts(logits, drafts, uniforms, draft_probs=draft_probs, temperature=temperature,
                                               counts=counts, lengths=lengths, **more)
    flag = kernels.device_status()
    assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in zip(before, (logits, drafts, uniforms)))
    heats = temperature.tolist() if isinstance(temperature, torch.Tensor) else [1.0 if temperature is None else temperature] * seqs
    # 256 threads a row at least add up their share one by one; 64 steps for the exponentials' arguments and approximation
    # and the joins; the result's own rounding and the largest element's
    error = 2.0 ** -24 * (vocab / 256 + 64)
    skipped, refused = 0, False
    for s in range(seqs):
        count = rows - 1 if counts is None else int(counts[s])
        want = verify(host(logits[s]), drafts[s].tolist(), uniforms[s].tolist(), None if draft_probs is None else host(draft_probs[s]),
                      heats[s], count)
        refused |= want[3]
        if want[4][0] < 2 * error or want[4][1] < 1e-12:
            skipped += 1
            continue
        assert tokens[s].tolist() == want[0].tolist(), (s, want[1])
        assert int(accepted[s]) == want[1]
        got = logprobs[s].double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want[2]))
        assert np.nanmax(np.abs(got - want[2]) - 2.0 ** -23 * np.abs(want[2])) <= error
        assert int(lengths[s]) == 100 + s - (min(max(count, 0), rows - 1) - want[1])
    assert skipped <= unclear, f"{skipped} sequences at a border"
    assert bool(flag & BAD) == refused or skipped
    return tokens, accepted, logprobs


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("probs", [*TYPES, None])
@pytest.mark.parametrize("seqs,n,vocab", [(3, 4, 1000), (9, 1, 50257), (2, 15, 4099), (40, 3, 515)])
def test_types_and_sizes(dtype, probs, seqs, n, vocab):
    need_gpu()
    check(*inputs(seqs, n, vocab, dtype=dtype, probs=probs, seed=vocab + n))


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 33, 255, 257, 2047, 151936, 262147])
def test_vocabularies(vocab):
    need_gpu()
    check(*inputs(5, 2, vocab, seed=vocab))
    check(*inputs(3, 3, vocab, seed=vocab + 1, dtype=torch.float32, probs=None))


@pytest.mark.parametrize("vocab,dtype,probs", [(3_000_001, torch.float32, torch.bfloat16), (5_000_003, torch.bfloat16, torch.float32),
                                               (2_100_000, torch.float16, None)])
def test_the_largest_vocabularies(vocab, dtype, probs):
    need_gpu()
    for near in (0.0, 0.7):
        check(*inputs(2, 1, vocab, seed=vocab, dtype=dtype, probs=probs, near=near))


def test_the_most_sequences():
    need_gpu()
    seqs, vocab = 65535, 9
    gen = torch.Generator(device="cuda").manual_seed(4)
    logits, uniforms = torch.randn(seqs, 1, vocab, generator=gen, device="cuda"), torch.rand(seqs, 1, generator=gen, device="cuda")
    none = torch.empty(seqs, 0, device="cuda", dtype=torch.int32)
    tokens, accepted, _ = verify_drafts(logits, none, uniforms)
    p = torch.softmax(logits[:, 0].double(), -1).cumsum(-1)
    target = uniforms.double() * p[:, -1:]
    clear = ((p - target).abs() > 1e-12).all(-1)
    assert torch.equal(tokens[clear, 0].long(), (p <= target).sum(-1)[clear]) and clear.sum() > seqs - 10 and (accepted == 0).all()
    with pytest.raises(ValueError, match="65535 sequences"):
        verify_drafts(torch.zeros(65536, 1, 8, device="cuda"), none.new_empty((65536, 0)), torch.zeros(65536, 1, device="cuda"))
    check(*inputs(600, 1, 100, seed=5))  # one CTA a sequence


@pytest.mark.parametrize("n", [0, 1, 15, 16, 31])
@pytest.mark.parametrize("seqs", [1, 7])
def test_numbers_of_drafts(n, seqs):
    need_gpu()
    # drafts from the target itself nearly always stay: every length of the accepted run is met
    for near in (0.0, 0.3):
        check(*inputs(seqs, n, 3001, seed=n, near=near, dtype=torch.float32))


def test_many_sequences_of_unequal_counts_and_temperatures():
    need_gpu()
    seqs, n = 300, 5
    heat = torch.tensor([(0.0, 0.3, 1.0, 1.7, 40.0)[i % 5] for i in range(seqs)], device="cuda")
    counts = torch.tensor([(i * 7) % (n + 1) for i in range(seqs)], device="cuda", dtype=torch.int32)
    logits, drafts, uniforms, probs = inputs(seqs, n, 2049, heat=heat, seed=5)
    # what lies behind the counts is not read
    behind = torch.arange(n + 1, device="cuda")[None] > counts[:, None]
    logits[behind] = math.nan
    probs[behind[:, 1:]] = math.nan
    drafts[behind[:, 1:]] = -5
    _, accepted, _ = check(logits, drafts, uniforms, probs, heat, counts)
    assert set(accepted.tolist()) == set(range(n + 1))
    check(logits, drafts.int(), uniforms, None, heat, counts)


def test_greedy_takes_the_lowest_of_equals():
    need_gpu()
    vocab, n = 5000, 3
    logits = torch.zeros(4, n + 1, vocab, device="cuda", dtype=torch.bfloat16)
    for j, at in enumerate(([4999], [17, 18, 4000], [0, 4999], [2500, 2501])):
        logits[:, j, at] = 3.0
    drafts = torch.tensor([[4999, 17, 0], [4999, 18, 0], [1, 17, 0], [4999, 17, 4999]], device="cuda")
    uniforms = torch.rand(4, n + 1, device="cuda")
    tokens, accepted, _ = check(logits, drafts, uniforms, None, 0.0)
    assert accepted.tolist() == [3, 1, 0, 2] and tokens.tolist() == [[4999, 17, 0, 2500], [4999, 17, -1, -1], [4999, -1, -1, -1], [4999, 17, 0, -1]]
    flat = torch.zeros(2, 1, 70001, device="cuda")
    assert check(flat, drafts[:2, :0], uniforms[:2, :1], None, 0.0)[0].tolist() == [[0], [0]]


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_tokens_have_no_probability(dtype):
    """-inf for all but a few tokens (a top-k filter), in whole parts of the row and at its ends; the type's lowest value too."""

    need_gpu()
    seqs, n, vocab = 24, 3, 9001
    logits, drafts, uniforms, probs = inputs(seqs, n, vocab, dtype=dtype, seed=2)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for s in range(seqs):
        keep = torch.randint(0, vocab, (1 + s % 4,), generator=gen, device="cuda")
        mask = torch.full((n + 1, vocab), -math.inf if s % 3 else torch.finfo(dtype).min, device="cuda", dtype=dtype)
        mask[:, keep] = logits[s][:, keep]
        logits[s] = mask
        if s % 2:
            drafts[s] = keep[0]
    for q in (probs, None):
        tokens, _, _ = check(logits, drafts, uniforms, q)
        chosen = logits.gather(2, tokens.clamp(min=0).long()[..., None])[..., 0]
        assert (chosen[tokens >= 0] > torch.finfo(dtype).min).all()


def test_rows_without_a_distribution():
    need_gpu()
    seqs, n, vocab = 9, 3, 3333
    for greedy in (False, True):
        logits, drafts, uniforms, _ = inputs(seqs, n, vocab, dtype=torch.float32, probs=None, seed=9)
        drafts[:] = logits[:, :n].argmax(-1)
        logits.scatter_(2, torch.cat((drafts, drafts[:, :1]), 1)[..., None], 60.0)  # certain: the drafts stay
        uniforms *= 0.9
        logits[1, 0, 5] = math.nan
        logits[2, 2, 3332] = math.nan
        logits[3, n, 0] = math.inf
        logits[4, 1] = -math.inf
        logits[5, 0] = math.nan
        logits[6, n] = -math.inf
        logits[7, 1, 100:3000] = -math.inf
        tokens, accepted, logprobs = check(logits, drafts, uniforms, None, 0.0 if greedy else None)
        masked = 1 if 100 <= int(drafts[7, 1]) < 3000 else 3  # a mask that takes the draft's probability, and no more
        assert accepted.tolist() == [3, 0, 2, 3, 1, 0, 3, masked, 3]
        assert [int(t[a]) < 0 for t, a in zip(tokens.tolist(), accepted.tolist())] == [False, True, True, True, True, True, True, False, False]
    # a NaN in the distribution that a draft was drawn from
    logits, drafts, uniforms, probs = inputs(3, 2, 100, seed=4)
    probs[1, 0] = math.nan
    tokens, accepted, _ = check(logits, drafts, uniforms, probs)
    assert tokens[1].tolist() == [-1, -1, -1] and int(accepted[1]) == 0


def test_drafts_outside_the_vocabulary_fall():
    need_gpu()
    logits, drafts, uniforms, probs = inputs(6, 3, 777, seed=8, near=0.0, dtype=torch.float32)
    drafts[0, 0], drafts[1, 1], drafts[2, 2], drafts[3, 0] = -1, 777, 1 << 30, -(1 << 31)
    check(logits, drafts.int(), uniforms, probs)
    drafts[4, 0], drafts[5, 1] = 1 << 40, -(1 << 40)  # 64 bits that 32 would cut to a token
    _, accepted, _ = check(logits, drafts, uniforms, probs)
    assert accepted.tolist()[0] == 0 and accepted.tolist()[4] == 0 and all(a <= 2 for a in accepted.tolist()[:3])
    check(logits, drafts, uniforms, None)


def test_counts_outside_are_limited():
    need_gpu()
    logits, drafts, uniforms, probs = inputs(4, 3, 500, seed=3)
    check(logits, drafts, uniforms, probs, None, torch.tensor([3, 9, -2, 1], device="cuda", dtype=torch.int32))


def test_random_numbers_at_their_ends():
    need_gpu()
    logits, drafts, uniforms, probs = inputs(8, 3, 601, seed=6, dtype=torch.float32)
    most = 1.0 - 2.0 ** -24
    uniforms[:4], uniforms[4:] = 0.0, most
    logits[1, 0] = -math.inf
    logits[1, 0, 600] = 1.0  # only the last token
    drafts[1, 0] = 600
    logits[2, 0, drafts[2, 0]] = -math.inf  # u = 0 does not take a token without probability
    logits[5, :, :7] = logits[5, :, 590:] = -math.inf
    for q in (probs, None):
        _, accepted, _ = check(logits, drafts, uniforms, q)
        assert accepted.tolist()[0] == 3 and accepted.tolist()[2] == 0


def test_nothing_left_of_the_target_falls_back_to_it():
    need_gpu()
    logits, drafts, uniforms, _ = inputs(6, 2, 2500, seed=7, dtype=torch.float32)
    probs = 3.0 * torch.softmax(logits[:, :2].double(), -1).float()  # more than the target everywhere
    uniforms[:, :2] = 0.9
    _, accepted, _ = check(logits, drafts, uniforms, probs)
    assert accepted.tolist() == [0] * 6
    one = torch.full((3, 2, 64), -math.inf, device="cuda")
    one[:, :, 9] = 0.0
    uniforms = torch.tensor([[0.5, 0.5]] * 3, device="cuda")
    half = torch.zeros(3, 1, 64, device="cuda")
    half[:, :, 9] = 2.5
    _, accepted, _ = check(one, torch.full((3, 1), 9, device="cuda"), uniforms, half)  # 0.5 * 2.5 is above 1
    assert accepted.tolist() == [0] * 3


@pytest.mark.parametrize("vocab", [257, 5000, 151936])
def test_draft_distributions_that_are_the_target_but_for_a_few_tokens(vocab):
    """Most of max(p - q, 0) is then rounding of q, on one side of the border or the other: the draw is over that as well."""

    need_gpu()
    seqs, n = 12, 1
    logits, drafts, uniforms, _ = inputs(seqs, n, vocab, seed=vocab, dtype=torch.float32, probs=None)
    p = torch.softmax(logits[:, :1].double(), -1)
    q = p.float()
    for s in range(seqs):
        order = p[s, 0].argsort(descending=True)
        a, b = int(order[0]), int(order[1 + 20 * (s % 4)])
        q[s, 0, a], q[s, 0, b] = p[s, 0, b], p[s, 0, a]  # offered far too often
        drafts[s, 0] = b
    uniforms[:, 0] = 1.0 - 2.0 ** -24
    _, accepted, _ = check(logits, drafts, uniforms, q)
    assert accepted.tolist() == [0] * seqs
    for s in range(seqs):  # and nothing but rounding: only the draft is offered a little too often
        q[s] = p[s].float()
        q[s, 0, drafts[s, 0]] *= 1.0 + 2.0 ** -18
    uniforms[:, 1] = torch.linspace(0.01, 0.99, seqs, device="cuda")
    tokens, accepted, _ = verify_drafts(logits, drafts, uniforms, draft_probs=q)
    for s in range(seqs):
        left = (p[s, 0] - q[s, 0].double()).clamp(min=0)
        if int(accepted[s]) == 0 and float(left.sum()) > 0:
            # p itself, in 64 bits, is off by 2^-52 of it: as much as 2^-27 of what rounding left
            running = left.cumsum(0) / left.sum()
            token, u = int(tokens[s, 0]), float(uniforms[s, 1])
            assert left[token] > 0 and float(running[token]) >= u - 1e-6 and float(running[token] - left[token] / left.sum()) <= u + 1e-6


@pytest.mark.parametrize("probs", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [3000, 151936])
def test_draft_distributions_that_are_the_target_rounded(probs, vocab):
    """Some elements are so near to p that they count for one side or the other by what Z is in its last bits."""

    need_gpu()
    seqs, n = 16, 1
    logits, drafts, uniforms, _ = inputs(seqs, n, vocab, seed=vocab, dtype=torch.float32, probs=None)
    heat = torch.linspace(0.4, 2.0, seqs, device="cuda")
    q = torch.softmax(logits[:, :1].double() / heat.double()[:, None, None], -1).to(probs)
    # of the drafts that are offered too often, the likeliest: with the largest random number it falls
    over = q.double() - torch.softmax(logits[:, :1].double() / heat.double()[:, None, None], -1)
    drafts[:] = over.argmax(-1)
    uniforms[:, 0] = 1.0 - 2.0 ** -24
    _, accepted, _ = check(logits, drafts, uniforms, q, heat, unclear=1)
    assert int(accepted.sum()) == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits_and_temperatures(dtype):
    need_gpu()
    logits, drafts, uniforms, _ = inputs(6, 2, 4000, dtype=torch.float32, probs=None, seed=11)
    big = (logits * (1000.0 if dtype is not torch.float16 else 400.0)).to(dtype)
    heat = torch.tensor([1.0, 0.01, 1000.0, 300.0, 1e-6, 1e6], device="cuda")
    check(big, drafts, uniforms, None, heat)
    check((logits + 20000.0).to(dtype), drafts, uniforms, None, heat)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_the_lowest_value_are_uniform(dtype):
    """A mask of the type's lowest value that leaves nothing; -inf beside it still has no probability."""

    need_gpu()
    vocab = 700
    logits = torch.full((40, 2, vocab), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    logits[20:, :, 10:] = -math.inf
    drafts = torch.full((40, 1), 3, device="cuda")
    uniforms = torch.rand(40, 2, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for heat in (None, 0.2, 30.0, 0.0):
        tokens, _, _ = check(logits, drafts, uniforms, None, heat)
        assert (tokens[20:] < 10).all()


def test_temperatures_at_their_ends():
    need_gpu()
    logits, drafts, uniforms, _ = inputs(8, 2, 900, seed=21, dtype=torch.float32, probs=None)
    logits[:, :, 100:300] = -math.inf
    heat = torch.tensor([1e-38, 1e-45, 1e30, 3e38, math.inf, 1e-30, -1.0, 1e-20], device="cuda")
    tokens, _, _ = check(logits[:4], drafts[:4], uniforms[:4], None, heat[:4].clamp(1e-30, 1e30))
    got = verify_drafts(logits, drafts, uniforms, temperature=heat)
    assert torch.equal(got[0][:4], tokens)
    masked = (got[0] >= 100) & (got[0] < 300)
    assert not masked.any() and kernels.device_status() == 0
    best = logits.argmax(-1)
    for s in (0, 1, 5, 6, 7):  # as good as greedy: the next token is the arg max of what is left
        at = int(got[1][s])
        left = logits[s, at].clone()
        if at < 2 and s != 6:
            left[drafts[s, at]] = -math.inf
        assert int(got[0][s, at]) == int(left.argmax()) and (at == 0 or int(got[0][s, 0]) == int(best[s, 0]))
    got = verify_drafts(logits, drafts, uniforms, temperature=torch.full((8,), math.nan, device="cuda"))
    assert (got[0][:, 0] == -1).all() and kernels.device_status() == BAD


def test_strides_alignment_and_shared_rows():
    need_gpu()
    seqs, n, vocab = 5, 3, 1001
    logits, drafts, uniforms, probs = inputs(seqs, n, vocab, seed=12)
    want = check(logits, drafts, uniforms, probs)
    for offset in (1, 3, 8):
        wide = torch.full((seqs, n + 1, vocab + 20), 100.0, device="cuda", dtype=logits.dtype)
        wide_q = torch.full((seqs, n, vocab + 20), 100.0, device="cuda")
        wide[..., offset:offset + vocab], wide_q[..., offset:offset + vocab] = logits, probs
        by_row = torch.zeros(n + 1, seqs, vocab, device="cuda", dtype=logits.dtype).copy_(logits.transpose(0, 1)).transpose(0, 1)
        pad = torch.zeros(seqs, n + 6, device="cuda", dtype=drafts.dtype)
        pad[:, 2:n + 2] = drafts
        u = torch.zeros(seqs, n + 9, device="cuda")
        u[:, :n + 1] = uniforms
        for x in (wide[..., offset:offset + vocab], by_row):
            got = verify_drafts(x, pad[:, 2:n + 2], u[:, :n + 1], draft_probs=wide_q[..., offset:offset + vocab])
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one target row and one distribution for all
    check(logits[:1, :1].expand(seqs, n + 1, vocab), drafts, uniforms, probs[:1, :1].expand(seqs, n, vocab))


def test_tokens_are_distributed_as_the_target():
    """4096 pairs of draft and draw: every token's frequency within five standard deviations of its probability."""

    need_gpu()
    seqs, vocab = 4096 * 8, 6
    gen = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn(1, 2, vocab, generator=gen, device="cuda")
    q = torch.softmax(torch.randn(1, 1, vocab, generator=gen, device="cuda"), -1)
    drafts = torch.multinomial(q[0, 0], seqs, replacement=True, generator=gen).view(seqs, 1)
    uniforms = torch.rand(seqs, 2, generator=gen, device="cuda")
    p = torch.softmax(logits[0, 0].double(), -1)
    for heat in (1.0, 0.5):
        p = torch.softmax(logits[0, 0].double() / heat, -1)
        tokens, accepted, _ = verify_drafts(logits.expand(seqs, 2, vocab), drafts, uniforms, draft_probs=q.expand(seqs, 1, vocab),
                                            temperature=heat)
        seen = torch.bincount(tokens[:, 0].long(), minlength=vocab).double()
        assert ((seen - seqs * p).abs() <= 5 * (seqs * p * (1 - p)).sqrt()).all()
        after = torch.bincount(tokens[accepted == 1, 1].long(), minlength=vocab).double()
        kept, p1 = int((accepted == 1).sum()), torch.softmax(logits[0, 1].double() / heat, -1)
        assert ((after - kept * p1).abs() <= 5 * (kept * p1 * (1 - p1)).sqrt()).all()


def test_captured_and_on_another_stream():
    need_gpu()
    logits, drafts, uniforms, probs = inputs(7, 4, 5003, seed=13)
    lengths = torch.full((7,), 1000, device="cuda", dtype=torch.int32)
    first = verify_drafts(logits, drafts, uniforms, draft_probs=probs, lengths=lengths)
    assert torch.equal(lengths, 1000 - (4 - first[1]))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = verify_drafts(logits, drafts, uniforms, draft_probs=probs)
        with torch.cuda.graph(graph, stream=stream):
            captured = verify_drafts(logits, drafts, uniforms, draft_probs=probs, lengths=lengths)
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (13, 14, 15):
        for x, y in zip((logits, drafts, uniforms, probs), inputs(7, 4, 5003, seed=seed)):
            x.copy_(y)
        lengths.fill_(50)
        graph.replay()
        want = verify_drafts(logits, drafts, uniforms, draft_probs=probs)
        assert all(torch.equal(a, b) for a, b in zip(captured, want)) and torch.equal(lengths, 50 - (4 - want[1]))
        if seed == 13:
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, again, captured))


def test_bad_calls_are_refused():
    need_gpu()
    logits, drafts, uniforms, probs = inputs(3, 2, 64, seed=1)
    fine = dict(draft_probs=probs)
    for change in (dict(logits=logits[0]), dict(logits=logits.double()), dict(logits=logits.transpose(1, 2).contiguous().transpose(1, 2)),
                   dict(drafts=drafts[:, :1]), dict(drafts=drafts.float()), dict(drafts=drafts.cpu()), dict(drafts=drafts.t().contiguous().t()),
                   dict(uniforms=uniforms[:, :2]), dict(uniforms=uniforms.double()), dict(draft_probs=probs[:, :1]),
                   dict(draft_probs=probs.double()), dict(draft_probs=probs.transpose(1, 2).contiguous().transpose(1, 2)),
                   dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
                   dict(temperature=torch.ones(2, device="cuda")), dict(temperature=torch.ones(3)),
                   dict(counts=torch.ones(3, device="cuda")), dict(counts=torch.ones(2, device="cuda", dtype=torch.int32)),
                   dict(lengths=torch.ones(3, device="cuda", dtype=torch.int64))):
        with pytest.raises(ValueError):
            args = {"logits": logits, "drafts": drafts, "uniforms": uniforms, **fine, **change}
            verify_drafts(args.pop("logits"), args.pop("drafts"), args.pop("uniforms"), **args)
    with pytest.raises(RuntimeError):
        verify_drafts(logits.cpu(), drafts, uniforms)
    with pytest.raises(ValueError, match="31 drafts"):
        verify_drafts(torch.zeros(1, 33, 8, device="cuda"), torch.zeros(1, 32, device="cuda", dtype=torch.int32), torch.zeros(1, 33, device="cuda"))
    none = verify_drafts(logits[:0], drafts[:0], uniforms[:0])
    assert [tuple(x.shape) for x in none] == [(0, 3), (0,), (0, 3)]
    assert kernels.device_status() == 0
