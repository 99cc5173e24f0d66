"""Attention over the 8-bit block cache at logits of any size: what the weights say must not
depend on how large the logits are that they come from."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from unicache_b200 import kernels

from .gpu_util import host, need_gpu
from .test_block8_gpu import HALF_ULP, make_cache, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[1, 2, 64, 700], [1, 5000, 333, 17000]])
@pytest.mark.parametrize("dim,block,queries,dtype", [(128, 64, 1, torch.bfloat16), (128, 16, 1, torch.float16),
                                                     (128, 64, 4, torch.float16), (64, 32, 1, torch.float16),
                                                     (64, 64, 4, torch.bfloat16)])
@pytest.mark.parametrize("size", [1.0, 1e4, 1e5, 1e6, 1e7])
def test_equal_logits_weigh_equally_whatever_their_size(size, dim, block, queries, dtype, lengths):
    """Each key is one row k of its head or zero, so a query's logits are one number or 0, bit for bit
    equal between tokens, and the output is the mean of the values with the larger one.  The weights
    are then equal: what is left of the errors is the fp16 rounding of a weight times its block's value scale
    (2^-11 relative, doubled) and 2^-17 for logarithm, exponentials and the fp32 sums."""

    need_gpu()
    heads, group, scale = 2, 5, 1.0
    cache, gen = make_cache(lengths, heads=heads, dim=dim, block=block, dtype=dtype, seed=3)
    total = sum(lengths)
    row = torch.randn(heads, dim, generator=gen, device="cuda").to(dtype)
    token = torch.cat([torch.arange(n, device="cuda") for n in lengths])
    key = torch.where((token % 3 == 1)[:, None, None], torch.zeros_like(row), row)
    # value scales that no power of two relates
    factor = 0.3 + 2.7 * torch.rand(total // 16 + 1, heads, 1, generator=gen, device="cuda")
    value = (torch.randn(total, heads, dim, generator=gen, device="cuda") * factor.repeat_interleave(16, 0)[:total]).to(dtype)
    cache.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    cache.write(key, value, starts=starts_of(lengths))
    restored_key, restored = (host(x).astype(np.float64) for x in restore(cache, lengths))
    # query heads along k, in turn with and against it; the last ones 1.5 times as large
    amount = size / float((row.float() ** 2).sum(-1).mean())
    if dtype is torch.float16:  # the rest by the scale of the softmax
        scale = max(1.0, amount / 4096)
        amount /= scale
    signs = torch.tensor([1.0, -1.0, 1.5, -1.5, 1.2], device="cuda")
    query = (row.float()[:, None] * signs[None, :, None] * amount).to(dtype).view(1, 1, heads * group, dim)
    query = query.expand(len(lengths), queries, -1, -1).contiguous()
    out, lse = cache.attention(query, softmax_scale=scale)
    got, got_lse, q = host(out).astype(np.float64), host(lse).astype(np.float64), host(query).astype(np.float64)
    at = 0
    for s, n in enumerate(lengths):
        zero = np.arange(n) % 3 == 1
        for i in range(queries):
            seen = np.arange(n) < n - queries + 1 + i
            for h in range(heads * group):
                if not seen.any():
                    assert np.isneginf(got_lse[s, i, h]) and (got[s, i, h] == 0).all()
                    continue
                logits = restored_key[at:at + n, h // group][seen] @ q[s, i, h] * scale
                p = np.exp(logits - logits.max())
                if size > 1:  # one of the two logits is all there is
                    assert set(np.round(p, 6)) <= {0.0, 1.0}
                v = restored[at:at + n, h // group][seen]
                expect, mean = p @ v / p.sum(), p @ np.abs(v) / p.sum()
                bound = np.abs(expect) * HALF_ULP[dtype] * 1.01 + mean * (2.0 ** -10 + 2.0 ** -17) + 2.0 ** -25
                if size <= 1:  # weights of two sizes: the logits' own error counts
                    bound = bound + mean * 2 * (dim + 8) * 2.0 ** -24 * (np.abs(q[s, i, h]) @ np.abs(host(row)[h // group])) * scale
                off = np.abs(got[s, i, h] - expect) - bound
                assert (off <= 0).all(), (size, n, i, h, float(off.max()))
                worst = np.abs(q[s, i, h]) @ np.abs(host(row)[h // group]) * scale
                at_most = (dim + 8) * 2.0 ** -24 * worst * 1.02 + 2.0 ** -20 + np.abs(logits.max()) * 2.0 ** -23
                assert abs(got_lse[s, i, h] - (logits.max() + np.log(p.sum()))) <= at_most
        at += n
    assert kernels.device_status() == 0


def restore(cache, lengths):
    """The codes times their scales in fp32 (rounded once more by the product, 2^-24)."""

    sides = []
    table = cache.block_table.long()
    for code, scale in ((cache.key_code, cache.key_scale), (cache.value_code, cache.value_scale)):
        rows = []
        for s, n in enumerate(lengths):
            pages = table[s, :-(-n // cache.block_size)]
            x = code[pages].float() * scale[pages][..., None, None]
            rows.append(x.transpose(1, 2).flatten(0, 1)[:n])
        sides.append(torch.cat(rows))
    return sides
