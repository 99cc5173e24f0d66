"""Seeded builders of the benchmark configurations' caches, assembled through
the public API (the same calls an engine makes), shared by ``bench.py`` and
the parity tests.

Config 4 (an image-editing layer, the shape the reference's long-query patch
targets, unicache/adapters/bagel.py:1598-1858): 28 query / 4 KV heads,
head_dim 128, bf16 K, V ~ N(0, 1) with 4 outlier key channels x10.  The cache
holds 256 instruction tokens and 4900 ViT tokens, each compressed by H2O to
20% (51 and 980 per KV head, scored by the attention of the current 1024-token
latent block over the full dense cache: the reference's "full_kv_first_call"
observation, operators/physical.py:51-101), 1024 source-VAE tokens in 2-bit
KIVI, group 32, with a 32-token bf16 residual (992 packed), and 16 boundary
tokens in bf16; the latent block's own 1024 keys/values stay dense.  The
query is the latent block: Lq = 1024 positions x 28 heads.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import kernels
from .adapters.attention import int8_block_decode, long_query_attention_summary, sparse_int8_block_decode
from .storage.block_pool import BlockPool
from .storage.int8_block import Int8BlockCache
from .storage.physical import GQAH2OCache, PackedKIVICache
from .synthetic import make_kv, make_query

CONFIG4 = {"instruction": 256, "vit": 4900, "vae": 1024, "boundary": 16, "latent": 1024, "lq": 1024,
           "q_heads": 28, "kv_heads": 4, "head_dim": 128, "ratio": 0.2, "recent_fraction": 0.25,
           "bits": 2, "group": 32, "residual": 32}


def h2o_budget(tokens: int, ratio: float, recent_fraction: float) -> tuple[int, int]:
    """(target, recent) per KV head, as the reference's storage backend
    computes them (Python rounding, tensor_backend.py:199-210)."""

    target = max(1, int(round(tokens * ratio)))
    return target, int(round(target * recent_fraction))


@dataclass
class Config4Layer:
    query: torch.Tensor            # [Lq, Hq, D] bf16
    dense: dict                    # name -> (key, value) [N, Hkv, D] bf16, the raw segments
    scores: dict                   # name -> [Hkv, N] fp32 H2O scores of the H2O segments
    first_call_lse: torch.Tensor   # [Hq, Lq] LSE of the latent block over the full dense cache
    segments: list                 # [instruction H2O, ViT H2O, VAE packed]
    dense_key: torch.Tensor        # boundary + latent rows [16 + 1024, Hkv, D]
    dense_value: torch.Tensor

    @property
    def key_tokens(self) -> int:
        n = int(self.dense_key.shape[0])
        for seg in self.segments:
            n += seg.retained_tokens if isinstance(seg, GQAH2OCache) else \
                seg.quantized_tokens + int(seg.residual_key.shape[0])
        return n


def config4_layer(device, seed: int = 1) -> Config4Layer:
    c = CONFIG4
    hkv, d = c["kv_heads"], c["head_dim"]
    names = ("instruction", "vit", "vae", "boundary", "latent")
    dense = {name: make_kv(c[name], hkv, d, seed=seed * 10 + i, device=device) for i, name in enumerate(names)}
    query = make_query(c["lq"], c["q_heads"], d, seed=seed, device=device)
    # First call: the latent block attends to the whole dense cache; its LSE
    # drives the H2O scores of the instruction and ViT segments.
    full_k = torch.cat([dense[n][0] for n in names])
    full_v = torch.cat([dense[n][1] for n in names])
    _, lse = long_query_attention_summary(query, [], dense_key=full_k, dense_value=full_v)
    scale = 1.0 / math.sqrt(d)
    scores, segments = {}, []
    for name in ("instruction", "vit"):
        k, v = dense[name]
        scores[name] = kernels.h2o_scores(query, k, lse, kv_heads=hkv, softmax_scale=scale)
        target, recent = h2o_budget(c[name], c["ratio"], c["recent_fraction"])
        segments.append(GQAH2OCache.from_dense(k, v, logical_token_ids=torch.arange(c[name], device=device),
                                               token_type_id=1, per_kv_head_scores=scores[name],
                                               target_tokens=target, recent_tokens=recent, selection_frozen=True))
    vk, vv = dense["vae"]
    segments.append(PackedKIVICache.from_dense(vk, vv, logical_token_ids=torch.arange(c["vae"], device=device),
                                               token_type_id=3, k_bits=c["bits"], v_bits=c["bits"],
                                               group_size=c["group"], residual_length=c["residual"]))
    dense_key = torch.cat([dense["boundary"][0], dense["latent"][0]])
    dense_value = torch.cat([dense["boundary"][1], dense["latent"][1]])
    return Config4Layer(query, dense, scores, lse, segments, dense_key, dense_value)


# ---------------------------------------------------------------- config 5
QWEN2_7B = {"hidden": 3584, "layers": 28, "q_heads": 28, "kv_heads": 4, "head_dim": 128, "ffn": 18944,
            "vocab": 151936, "rope_theta": 1.0e6, "eps": 1.0e-6}


class Qwen2PackedDecode:
    """a Qwen2-7B-shaped decoder (hidden 3584, 28 layers, 28
    query / 4 KV heads, head_dim 128, FFN 18944, untied 151936-token head:
    modeling/qwen2/configuration_qwen2.py:123-134 of the reference) with
    seeded random bf16 weights, decoding ``batch`` sequences greedily.

    Each layer's prompt cache of ``prompt`` tokens per sequence is synthetic
    (seeded K/V with the benchmark's distribution and seeded H2O scores, in
    place of a prefill), compressed by H2O to ``ratio`` of the tokens per KV
    head (the reference's recent fraction 0.25) and the retained rows packed
    in ``bits``-bit KIVI (group ``group``, ``residual`` bf16 tokens) -- the
    composition the reference refuses on one request (tensor_backend.py:
    137-144) applied as two steps.  New tokens go to a dense bf16 suffix of
    capacity ``new_tokens`` (the reference appends decode tokens to its dense
    cache).  Attention is the packed decode kernel over [packed prompt +
    residual + live suffix]; the projections are cuBLAS GEMMs through torch
    (residual adds in their epilogues), and RMSNorm, the rotary embedding
    fused with the suffix append, and the SwiGLU gate are one library kernel
    each (``kernels.rms_norm``, ``qkv_rope_append``, ``silu_mul``): ten
    launches per layer.  One decode step is captured once as a CUDA graph:
    the suffix length, the RoPE position and the append index live on the
    device.
    """

    def __init__(self, device, *, batch: int = 32, prompt: int = 16384, new_tokens: int = 512,
                 ratio: float = 0.2, recent_fraction: float = 0.25, bits: int = 2, group: int = 32,
                 residual: int = 32, layers: int | None = None, prefilled: int = 0, seed: int = 5):
        from .kernels import GrowingSuffix

        c = QWEN2_7B
        self.device = torch.device(device)
        self.batch, self.prompt, self.capacity = batch, prompt, new_tokens
        self.layers = c["layers"] if layers is None else layers
        hid, hq, hkv, d, ffn = c["hidden"], c["q_heads"], c["kv_heads"], c["head_dim"], c["ffn"]
        self.hq, self.hkv, self.d, self.ffn, self.eps = hq, hkv, d, ffn, c["eps"]
        gen = torch.Generator(device=self.device).manual_seed(seed)

        def weight(*shape, std=0.02):
            return (torch.randn(*shape, generator=gen, device=self.device) * std).to(torch.bfloat16)

        qkv_out = (hq + 2 * hkv) * d
        self.w = []
        for _ in range(self.layers):
            self.w.append({
                "in_norm": torch.ones(hid, device=self.device, dtype=torch.bfloat16),
                "qkv": weight(hid, qkv_out), "qkv_bias": weight(qkv_out),
                "o": weight(hq * d, hid),
                "post_norm": torch.ones(hid, device=self.device, dtype=torch.bfloat16),
                "gate_up": weight(hid, 2 * ffn), "down": weight(ffn, hid),
            })
        self.embed = weight(c["vocab"], hid)
        self.final_norm = torch.ones(hid, device=self.device, dtype=torch.bfloat16)
        self.lm_head = weight(hid, c["vocab"])
        half = d // 2
        self.inv_freq = 1.0 / (c["rope_theta"] ** (torch.arange(half, device=self.device, dtype=torch.float32) / half))

        # caches: H2O 20% of the prompt per KV head, then KIVI on the retained rows
        target, recent = h2o_budget(prompt, ratio, recent_fraction)
        self.retained = target
        self.length = torch.full((1,), prefilled, device=self.device, dtype=torch.int32)
        self.plans, self.suffixes, self.packed = [], [], []
        outliers = torch.randperm(d, generator=torch.Generator().manual_seed(seed))[:4].to(self.device)
        for layer in range(self.layers):
            sk = torch.zeros(batch, new_tokens, hkv, d, device=self.device, dtype=torch.bfloat16)
            sv = torch.zeros_like(sk)
            if prefilled:
                sk[:, :prefilled] = weight(batch, prefilled, hkv, d, std=1.0)
                sv[:, :prefilled] = weight(batch, prefilled, hkv, d, std=1.0)
            self.suffixes.append((sk, sv))
            seqs = []
            for b in range(batch):
                # generated on the device (the prompt caches are tens of GB in total)
                k = torch.randn(prompt, hkv, d, generator=gen, device=self.device)
                k[:, :, outliers] *= 10.0
                k = k.to(torch.bfloat16)
                v = torch.randn(prompt, hkv, d, generator=gen, device=self.device).to(torch.bfloat16)
                scores = torch.rand(hkv, prompt, generator=gen, device=self.device)
                kept = GQAH2OCache.from_dense(k, v, logical_token_ids=torch.arange(prompt, device=self.device),
                                              token_type_id=0, per_kv_head_scores=scores, target_tokens=target,
                                              recent_tokens=recent, selection_frozen=True)
                packed = PackedKIVICache.from_dense(kept.key.transpose(0, 1), kept.value.transpose(0, 1),
                                                    logical_token_ids=kept.logical_token_ids[0], token_type_id=0,
                                                    k_bits=bits, v_bits=bits, group_size=group,
                                                    residual_length=residual)
                del k, v, kept
                seqs.append([packed, GrowingSuffix(sk[b], sv[b], self.length)])
                self.packed.append(packed)
            from .kernels import build_decode_plan

            self.plans.append(build_decode_plan(seqs, num_kv_heads=hkv, head_dim=d))
        torch.cuda.empty_cache()
        self.ids = torch.zeros(batch, device=self.device, dtype=torch.int64)
        self.x = self.embed[self.ids].clone()
        self.q_buf = torch.empty(batch, hq, d, device=self.device, dtype=torch.bfloat16)
        self.attn_out = torch.empty(batch, hq, d, device=self.device, dtype=torch.bfloat16)
        self.attn_lse = torch.empty(batch, hq, device=self.device, dtype=torch.float32)
        self.graph = None

    # bytes one decode step must read: every weight matrix once (the embedding
    # gather is a few rows), the packed prompt of every layer and sequence,
    # and the live suffix rows.
    def weight_bytes(self) -> int:
        per_layer = sum(t.numel() * t.element_size() for t in self.w[0].values())
        return per_layer * self.layers + self.lm_head.numel() * 2 + self.final_norm.numel() * 2

    def cache_bytes(self, suffix_len: int) -> int:
        prompt = sum(p.bytes_per_step for p in self.plans)
        grown = self.layers * self.batch * self.hkv * self.d * 4 * suffix_len  # bf16 K and V rows
        capacity = self.layers * self.batch * self.hkv * self.d * 4 * self.capacity
        return prompt - capacity // 2 + grown  # the plans weight the suffix at half its capacity

    def step(self) -> torch.Tensor:
        """One greedy decode step of every sequence (device-only, capturable):
        returns the next token ids [batch]."""

        from . import kernels

        b, hq, hkv, d = self.batch, self.hq, self.hkv, self.d
        self.length += 1  # this step's token is row length - 1 of every suffix
        x = self.x
        for layer in range(self.layers):
            w = self.w[layer]
            h = kernels.rms_norm(x, w["in_norm"], self.eps)
            qkv = torch.addmm(w["qkv_bias"], h, w["qkv"])
            sk, sv = self.suffixes[layer]
            # rotary embedding, the query for the decode kernel, the key and
            # value appended to the suffix row the device-side length names
            kernels.qkv_rope_append(qkv, hq=hq, hkv=hkv, length=self.length, prompt=self.prompt,
                                    inv_freq=self.inv_freq, q_out=self.q_buf, suffix_k=sk, suffix_v=sv)
            self.plans[layer].run(self.q_buf, out=self.attn_out, lse=self.attn_lse)
            x = torch.addmm(x, self.attn_out.view(b, hq * d), w["o"])
            h = kernels.rms_norm(x, w["post_norm"], self.eps)
            x = torch.addmm(x, kernels.silu_mul(h @ w["gate_up"]), w["down"])
        logits = kernels.rms_norm(x, self.final_norm, self.eps) @ self.lm_head
        self.ids.copy_(torch.argmax(logits, dim=-1))
        self.x.copy_(self.embed[self.ids])
        return self.ids

    def capture(self) -> None:
        """Capture one decode step as a CUDA graph (after a first eager step has
        done every first-call set-up); ``replay`` then runs a step."""

        stream = torch.cuda.Stream(device=self.device)
        stream.wait_stream(torch.cuda.current_stream(self.device))
        self.graph = torch.cuda.CUDAGraph()
        saved = self.length.clone()
        with torch.cuda.stream(stream):
            with torch.cuda.graph(self.graph, stream=stream):
                self.step()
        torch.cuda.current_stream(self.device).wait_stream(stream)
        self.length.copy_(saved)  # capture does not run the step

    def replay(self) -> None:
        self.graph.replay()


# ---------------------------------------------------------------- decode over the 8-bit block cache
class Int8BlockDecode:
    """Attention layers with head norms decoding over 8-bit block caches.

    Each layer normalises its input, projects it, normalises and rotates the
    query and key heads (``head_norm_rope``), appends key and value to its
    ``Int8BlockCache`` and attends over the whole cache or, with ``count``,
    over that many blocks that the query chooses (``sparse_int8_block_decode``).
    All layers share one block table and one device tensor of lengths, so a
    step has no host state and is captured once as a CUDA graph.  Weights and
    prompts are seeded random; the prompts' keys go through the same norm and
    rotation and all sequences of a layer through one write.
    """

    def __init__(self, device, *, prompts: list[int], new_tokens: int, layers: int = 2, hidden: int = 3584,
                 q_heads: int = 28, kv_heads: int = 4, head_dim: int = 128, block_size: int = 64,
                 count: int | None = None, theta: float = 1.0e6, seed: int = 7):
        self.device = torch.device(device)
        self.hq, self.hkv, self.d, self.count, self.eps = q_heads, kv_heads, head_dim, count, 1.0e-6
        gen = torch.Generator(device=self.device).manual_seed(seed)

        def normal(*shape, std=1.0, mean=0.0):
            return (mean + std * torch.randn(*shape, generator=gen, device=self.device)).to(torch.bfloat16)

        batch, longest, tokens = len(prompts), max(prompts) + new_tokens, sum(prompts)
        self.cos, self.sin = kernels.rope_table(longest, head_dim, theta=theta, device=self.device)
        starts = torch.tensor([0, *prompts], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(self.device)
        where = torch.cat([torch.arange(n, dtype=torch.int32) for n in prompts]).to(self.device)
        self.w, self.caches = [], []
        for layer in range(layers):
            weights = {"norm": normal(hidden, std=0.1, mean=1.0),
                       "qkv": normal(hidden, (q_heads + 2 * kv_heads) * head_dim, std=hidden ** -0.5),
                       "q_norm": normal(head_dim, std=0.1, mean=1.0), "k_norm": normal(head_dim, std=0.1, mean=1.0),
                       "o": normal(q_heads * head_dim, hidden, std=hidden ** -0.5)}
            shared = {} if layer == 0 else {"block_table": self.caches[0].block_table,
                                            "num_blocks": int(self.caches[0].key_code.shape[0]),
                                            "lengths": self.caches[0].lengths}
            cache = Int8BlockCache.allocate(batch, longest, num_kv_heads=kv_heads, head_dim=head_dim,
                                            block_size=block_size, device=self.device, **shared)
            if layer == 0:
                cache.advance(torch.tensor(prompts, dtype=torch.int32, device=self.device))
            key, value = normal(tokens, kv_heads, head_dim), normal(tokens, kv_heads, head_dim)
            _, key = kernels.head_norm_rope(None, key, None, weights["k_norm"], self.cos, self.sin, where, eps=self.eps)
            cache.write(key, value, starts=starts)
            self.w.append(weights)
            self.caches.append(cache)
        self.x = normal(batch, hidden)
        self.query = self.attended = None  # the last layer's, of the last step
        self.graph = None

    def step(self) -> torch.Tensor:
        """One token of every sequence (device-only, capturable): the hidden states [batch, hidden]."""

        hq, hkv, d = self.hq, self.hkv, self.d
        lengths = self.caches[0].lengths
        self.caches[0].advance(1)  # for every layer
        positions = lengths - 1
        x = self.x
        for w, cache in zip(self.w, self.caches):
            qkv = (kernels.rms_norm(x, w["norm"], self.eps) @ w["qkv"]).view(-1, hq + 2 * hkv, d)
            query, key = kernels.head_norm_rope(qkv[:, :hq], qkv[:, hq:hq + hkv], w["q_norm"], w["k_norm"], self.cos,
                                                self.sin, positions, eps=self.eps)
            cache.write(key, qkv[:, hq + hkv:])
            if self.count is None:
                out, _ = int8_block_decode(query, cache)
            else:
                _, out, _ = sparse_int8_block_decode(query, cache, count=self.count)
            x = torch.addmm(x, out.view(-1, hq * d), w["o"])
        self.query, self.attended = query, out
        self.x.copy_(x)
        return self.x

    def capture(self) -> None:
        """Capture one step as a CUDA graph; ``replay`` then runs a step."""

        if self.query is None:  # a first step does every first-call set-up; its rows are withdrawn
            before = self.x.clone()
            self.step()
            self.caches[0].advance(-1)
            self.x.copy_(before)
        stream = torch.cuda.Stream(device=self.device)
        stream.wait_stream(torch.cuda.current_stream(self.device))
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            with torch.cuda.graph(self.graph, stream=stream):
                self.step()
        torch.cuda.current_stream(self.device).wait_stream(stream)

    def replay(self) -> torch.Tensor:
        self.graph.replay()
        return self.x


# ---------------------------------------------------------------- drafted decode over a pool of blocks
class DraftDecode:
    """A small decoder that verifies drafted tokens over 8-bit caches of one block pool.

    Every prompt starts with an image of ``image`` patches, whose keys turn by the time, row and column of the patch; text goes on behind
    it on all axes.  A prompt is written once and continued in ``samples`` sequences (``BlockPool.fork``).  A step draws
    ``drafts`` tokens a sequence from as many linear heads over the last hidden state, runs all of them through the
    layers at once (``head_norm_rope`` by axes, ``Int8BlockCache.write``, ``int8_block_decode`` with several query tokens) and keeps what
    ``verify_drafts`` leaves of them, which lowers the lengths that all layers share.  A draft that may be rejected in part
    must not go past the end of its block, so a sequence near it drafts fewer.  Blocks, counts and lengths are on
    the device: a step has no host state and is captured once as a CUDA graph.  Weights and prompts are seeded random.
    """

    def __init__(self, device, *, prompts: list[int], new_tokens: int, samples: int = 1, drafts: int = 3,
                 image: tuple[int, int] = (4, 6), layers: int = 2, hidden: int = 512, q_heads: int = 8, kv_heads: int = 2,
                 head_dim: int = 64, block_size: int = 64, vocab: int = 4096, temperature: float = 1.0, theta: float = 1.0e4,
                 seed: int = 11):
        self.device = torch.device(device)
        self.hq, self.hkv, self.d, self.eps, self.n, self.vocab = q_heads, kv_heads, head_dim, 1.0e-6, drafts, vocab
        patches, self.block = image[0] * image[1], block_size
        if min(prompts) <= patches or not 0 <= drafts < min(16, block_size):
            raise ValueError("prompts must be longer than the image, and drafts fewer than 16 and a block's tokens")
        gen = torch.Generator(device=self.device).manual_seed(seed)

        def normal(*shape, std=1.0, mean=0.0):
            return (mean + std * torch.randn(*shape, generator=gen, device=self.device, dtype=torch.float32)).to(torch.bfloat16)

        count, longest = len(prompts), max(prompts) + new_tokens + drafts + 1
        seqs = count * samples
        width = -(-longest // block_size)
        self.pool = BlockPool.allocate(seqs, longest, sum(-(-n // block_size) for n in prompts) + seqs * (width - min(prompts) // block_size),
                                       block_size=block_size, device=self.device)
        self.cos, self.sin = kernels.rope_table(longest, head_dim, theta=theta, device=self.device)
        half = head_dim // 2
        sections = [half // 4 // 4 * 4, half // 8 * 3, half - half // 4 // 4 * 4 - half // 8 * 3]
        self.axes = kernels.rope_axes(sections)
        # positions of a prompt's tokens: patches by row and column, then text from the larger of the two on
        i = torch.arange(longest, device=self.device, dtype=torch.int32)
        text = i - patches + max(image)
        self.where = torch.stack([torch.where(i < patches, x, text) for x in (i * 0, i // image[1], i % image[1])]).contiguous()
        rows = torch.cat([torch.arange(n) for n in prompts]).to(self.device)
        ends = torch.tensor([0, *prompts], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        starts = ends.tolist() + [ends[-1].item()] * (seqs - count)  # prompts in the first sequences
        starts = torch.tensor(starts, dtype=torch.int32, device=self.device)
        self.pool.advance(starts[1:] - starts[:-1])
        self.w, self.caches = [], []
        for _ in range(layers):
            weights = {"norm": normal(hidden, std=0.1, mean=1.0),
                       "qkv": normal(hidden, (q_heads + 2 * kv_heads) * head_dim, std=hidden ** -0.5),
                       "q_norm": normal(head_dim, std=0.1, mean=1.0), "k_norm": normal(head_dim, std=0.1, mean=1.0),
                       "o": normal(q_heads * head_dim, hidden, std=hidden ** -0.5)}
            cache = self.pool.cache(num_kv_heads=kv_heads, head_dim=head_dim)
            key, value = normal(sum(prompts), kv_heads, head_dim), normal(sum(prompts), kv_heads, head_dim)
            _, key = kernels.head_norm_rope(None, key, None, weights["k_norm"], self.cos, self.sin,
                                            self.where[:, rows].contiguous(), eps=self.eps, axes=self.axes)
            cache.write(key, value, starts=starts)
            self.w.append(weights)
            self.caches.append(cache)
        if samples > 1:
            children = torch.arange(count, seqs, dtype=torch.int32, device=self.device)
            self.pool.fork(children % count, children)
        self.embed, self.final_norm = normal(vocab, hidden), normal(hidden, std=0.1, mean=1.0)
        self.lm_head = normal(hidden, vocab, std=4.0 * hidden ** -0.5)
        # heads near the model's own, so that some drafts stay
        self.draft_heads = torch.cat([self.lm_head + normal(hidden, vocab, std=1.0 * hidden ** -0.5) for _ in range(drafts)], 1) \
            if drafts else None
        self.temperature = torch.full((seqs,), float(temperature), device=self.device, dtype=torch.float32)
        self.last = torch.randint(0, vocab, (seqs,), generator=gen, device=self.device, dtype=torch.int32)
        self.state = normal(seqs, hidden)  # of the token in front of the last one
        self.uniforms = torch.rand(seqs, 2 * drafts + 1, generator=gen, device=self.device, dtype=torch.float32)  # the caller's to renew
        self.graph = self.result = None

    def propose(self):
        """(drafts int32 [seqs, n], their distributions): one linear head each over the last hidden state."""

        seqs, n = self.last.shape[0], self.n
        if n == 0:
            return self.last.new_empty((seqs, 0)), None
        logits = (self.state @ self.draft_heads).view(seqs * n, 1, self.vocab)
        heat = self.temperature.repeat_interleave(n)
        # a draw without drafts to verify
        tokens, _, _ = kernels.verify_drafts(logits, self.last.new_empty((seqs * n, 0)),
                                             self.uniforms[:, :n].reshape(seqs * n, 1), temperature=heat)
        probs = torch.softmax(logits.float() / torch.where(heat > 0, heat, 1.0)[:, None, None], -1)
        return tokens.view(seqs, n), probs.view(seqs, n, self.vocab)

    def step(self):
        """One verified step of every sequence (device-only, capturable): (tokens [seqs, n + 1], accepted [seqs], logprobs)."""

        hq, hkv, d, n = self.hq, self.hkv, self.d, self.n
        lengths, seqs = self.pool.lengths, self.last.shape[0]
        drafts, probs = self.propose()
        held = lengths.clone()
        counts = torch.clamp(self.block - 1 - held % self.block, max=n).to(torch.int32)  # up to the block's end
        self.pool.advance(counts + 1)
        # rows of the last token and its drafts; those that count, one behind the other, are the write's
        i = torch.arange(n + 1, device=self.device)
        meant = i[None] <= counts[:, None]
        order = torch.sort((~meant).flatten().to(torch.uint8), stable=True).indices
        starts = torch.zeros(seqs + 1, dtype=torch.int32, device=self.device)
        torch.cumsum(counts + 1, 0, dtype=torch.int32, out=starts[1:])
        positions = self.where[:, torch.clamp(held[:, None] + i, max=self.where.shape[1] - 1).flatten()]
        # the attention takes a sequence's queries as its last tokens: rows that count to the end, and back
        gap = (n - counts)[:, None]
        to_end = (torch.clamp(i[None] - gap, min=0) + (n + 1) * torch.arange(seqs, device=self.device)[:, None]).flatten()
        back = (torch.clamp(i[None] + gap, max=n) + (n + 1) * torch.arange(seqs, device=self.device)[:, None]).flatten()
        x = self.embed[torch.cat((self.last[:, None], drafts), 1).flatten().long()]
        for w, cache in zip(self.w, self.caches):
            qkv = (kernels.rms_norm(x, w["norm"], self.eps) @ w["qkv"]).view(-1, hq + 2 * hkv, d)
            query, key = kernels.head_norm_rope(qkv[:, :hq], qkv[:, hq:hq + hkv], w["q_norm"], w["k_norm"], self.cos,
                                                self.sin, positions, eps=self.eps, axes=self.axes)
            cache.write(key[order], qkv[:, hq + hkv:][order], starts=starts)
            out, _ = int8_block_decode(query[to_end].view(seqs, n + 1, hq, d), cache)
            x = torch.addmm(x, out.view(-1, hq * d)[back], w["o"])
        x = kernels.rms_norm(x, self.final_norm, self.eps)
        logits = (x @ self.lm_head).view(seqs, n + 1, self.vocab)
        tokens, accepted, logprobs = kernels.verify_drafts(logits, drafts, self.uniforms[:, n:], draft_probs=probs,
                                                           temperature=self.temperature, counts=counts, lengths=lengths)
        at = accepted.long()[:, None]
        self.last.copy_(tokens.gather(1, at)[:, 0])
        self.state.copy_(x.view(seqs, n + 1, -1).gather(1, at[..., None].expand(-1, -1, x.shape[-1]))[:, 0])
        self.result = {"logits": logits, "drafts": drafts, "probs": probs, "counts": counts}
        return tokens, accepted, logprobs

    def finish(self, sequences: torch.Tensor) -> None:
        """Sequences (int32) that have ended: their blocks are free, and those still in use move together."""

        self.pool.release(sequences)
        self.pool.compact()

    def capture(self) -> None:
        """Capture one step as a CUDA graph, after a first eager one; ``replay`` then runs a step."""

        stream = torch.cuda.Stream(device=self.device)
        stream.wait_stream(torch.cuda.current_stream(self.device))
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            with torch.cuda.graph(self.graph, stream=stream):
                self.captured = self.step()
        torch.cuda.current_stream(self.device).wait_stream(stream)

    def replay(self):
        self.graph.replay()
        return self.captured
