"""The decode layer around the wave-index attention, with random-initialised weights.

Mirror of the reference's decode loop (model_hub/LLM.py:90-126 ``layer_decode``, :156-171
``decode_forward``) for measuring decode tokens/s with the projections and the MLP included.
There are no checkpoints here, so the weights are seeded Gaussians at the model's true shapes.
The projections are plain library GEMMs (``torch.nn.functional.linear``, as the reference); the
element-wise work between them runs in this package's kernels (``ri_rmsnorm`` with the residual
add folded in, ``ri_rope_split``, ``ri_silu_and_mul``); the attention is
``decode_update_kv_cache`` + ``compute`` of a ``retroinfer_cache``.

Every buffer is allocated once, positions live on the device, and nothing synchronises: one
decode step can be captured in a CUDA graph and replayed.

``PagedDecoder`` runs the same layers, prompts included, over a ``paged_cache``: positions may have several
axes (text, images, video), and requests of uneven lengths share a pool of pages and are held to a number of slots.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import _lib


@dataclass
class ModelShape:
    hidden: int
    intermediate: int
    vocab: int
    layers: int
    q_heads: int
    kv_heads: int
    head_dim: int = 128
    rope_theta: float = 5e5
    rms_eps: float = 1e-5

    @property
    def qkv_dim(self) -> int:
        return (self.q_heads + 2 * self.kv_heads) * self.head_dim


# published geometries of the models the benchmark configurations name
LLAMA3_8B = ModelShape(4096, 14336, 128256, 32, 32, 8, rope_theta=5e5, rms_eps=1e-5)
QWEN25_7B = ModelShape(3584, 18944, 152064, 28, 28, 4, rope_theta=1e6, rms_eps=1e-6)
QWEN25_72B = ModelShape(8192, 29568, 152064, 80, 64, 8, rope_theta=1e6, rms_eps=1e-6)


def rmsnorm(x, weight, eps, out, residual=None):
    """``out = rmsnorm(residual + x) * weight`` (``residual`` updated in place) or ``rmsnorm(x) * weight``."""
    rows, dim = x.shape
    _lib.check(_lib.lib.ri_rmsnorm(x.data_ptr(), _lib.ptr(residual), weight.data_ptr(), out.data_ptr(), rows, dim,
                                   float(eps), _lib.dtype_code(x.dtype), _lib.current_stream()), "ri_rmsnorm")
    return out


def rope_split(qkv, cos_sin, positions, q, k, v):
    """Rotate the query/key heads of ``qkv`` ``[rows, (Hq+2Hk)*128]`` at ``positions`` and split into ``q, k, v``."""
    rows, q_heads, kv_heads = q.shape[0], q.shape[-2], k.shape[-2]
    assert qkv.shape == (rows, (q_heads + 2 * kv_heads) * 128) and cos_sin.dtype == torch.float32
    assert cos_sin.shape[1] == 128 and positions.dtype == torch.int64 and positions.numel() == rows
    _lib.check(_lib.lib.ri_rope_split(qkv.data_ptr(), cos_sin.data_ptr(), positions.data_ptr(), q.data_ptr(),
                                      k.data_ptr(), v.data_ptr(), rows, q_heads, kv_heads, cos_sin.shape[0],
                                      _lib.dtype_code(qkv.dtype), _lib.current_stream()), "ri_rope_split")


def silu_and_mul(x, out):
    rows, two_inter = x.shape
    _lib.check(_lib.lib.ri_silu_and_mul(x.data_ptr(), out.data_ptr(), rows, two_inter // 2, _lib.dtype_code(x.dtype),
                                        _lib.current_stream()), "ri_silu_and_mul")
    return out


def cos_sin_cache(max_positions: int, head_dim: int, theta: float, device) -> torch.Tensor:
    """fp32 ``[max_positions, head_dim]``: cosines then sines (model_hub/llama.py:81-84, :109)."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim))
    freqs = torch.outer(torch.arange(max_positions, dtype=torch.float32, device=device), inv_freq)
    return torch.cat((freqs.cos(), freqs.sin()), dim=-1).contiguous()


class SyntheticDecoder:
    """Decode-only model with seeded random weights over a prepared ``retroinfer_cache``."""

    def __init__(self, shape: ModelShape, cache, batch: int, max_positions: int, device, dtype=torch.bfloat16,
                 seed: int = 0, std: float = 0.02, layers: int | None = None):
        self.shape, self.cache, self.batch, self.device, self.dtype = shape, cache, batch, device, dtype
        self.n_layers = shape.layers if layers is None else layers
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)

        def w(*s):
            return (torch.randn(s, generator=gen, device=device, dtype=torch.float32) * std).to(dtype)

        h, it = shape.hidden, shape.intermediate
        self.embed = w(shape.vocab, h)
        self.lm_head = w(shape.vocab, h)
        self.final_norm = torch.ones(h, dtype=dtype, device=device)
        self.layers = []
        for _ in range(self.n_layers):
            self.layers.append(dict(wqkv=w(shape.qkv_dim, h), wo=w(h, shape.q_heads * shape.head_dim),
                                    gate_up=w(2 * it, h), down=w(h, it),
                                    norm1=torch.ones(h, dtype=dtype, device=device),
                                    norm2=torch.ones(h, dtype=dtype, device=device)))
        self.cos_sin = cos_sin_cache(max_positions, shape.head_dim, shape.rope_theta, device)
        # the position of the token being decoded, per request (the reference slices position_ids at
        # kv_cache.context, model_hub/llama.py:330-337); advanced on the device after every step
        self.positions = torch.full((batch,), int(cache.context), dtype=torch.int64, device=device)
        z = lambda *s: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
        self.input_ids = torch.zeros((batch,), dtype=torch.int64, device=device)
        self.residual, self.normed = z(batch, h), z(batch, h)
        self.q = z(batch, 1, shape.q_heads, shape.head_dim)
        self.k = z(batch, 1, shape.kv_heads, shape.head_dim)
        self.v = z(batch, 1, shape.kv_heads, shape.head_dim)
        self.attn = z(batch, 1, shape.q_heads, shape.head_dim)
        self.act = z(batch, it)
        self.next_ids = torch.zeros((batch,), dtype=torch.int64, device=device)

    def layer_decode(self, ldx: int, x: torch.Tensor) -> torch.Tensor:
        """One layer (model_hub/LLM.py:90-126).  ``x`` is the previous block's output that has not been
        added to the residual stream yet (None for the first layer: the residual holds the embedding)."""
        s, L = self.shape, self.layers[ldx]
        rmsnorm(self.residual if x is None else x, L["norm1"], s.rms_eps, self.normed,
                residual=None if x is None else self.residual)
        qkv = F.linear(self.normed, L["wqkv"])
        rope_split(qkv, self.cos_sin, self.positions, self.q, self.k, self.v)
        self.cache.decode_update_kv_cache(self.k, self.v, ldx)
        # attn_hub.retroinfer_decode_attn is cache.compute; called directly to hand it the output buffer
        attn = self.cache.compute(self.q, ldx, out=self.attn)
        o = F.linear(attn.view(self.batch, -1), L["wo"])
        rmsnorm(o, L["norm2"], s.rms_eps, self.normed, residual=self.residual)
        silu_and_mul(F.linear(self.normed, L["gate_up"]), self.act)
        return F.linear(self.act, L["down"])

    def decode_forward(self) -> torch.Tensor:
        """One decode step for ``input_ids`` (model_hub/LLM.py:156-171): logits ``[batch, vocab]`` fp32;
        the greedy next ids are left in ``next_ids`` and become ``input_ids`` of the next step."""
        torch.index_select(self.embed, 0, self.input_ids, out=self.residual)
        x = None
        for ldx in range(self.n_layers):
            x = self.layer_decode(ldx, x)
        rmsnorm(x, self.final_norm, self.shape.rms_eps, self.normed, residual=self.residual)
        logits = F.linear(self.normed, self.lm_head).float()
        torch.argmax(logits, dim=-1, out=self.next_ids)
        self.input_ids.copy_(self.next_ids)
        self.positions.add_(1)
        return logits

    def weight_bytes_per_step(self) -> int:
        """Bytes of weights one decode step reads (every matrix once; one embedding row per request)."""
        per_layer = sum(t.numel() * t.element_size() for t in self.layers[0].values())
        return per_layer * self.n_layers + self.lm_head.numel() * self.lm_head.element_size()


class PagedDecoder(SyntheticDecoder):
    """The same model over a ``paged_cache``: prompts of uneven lengths in one pass, then a token of every running request a step.
    A request that is done gives its place back (``release``), and another prompt may take it while the rest run on.  ``axis_of``: the position axis of each rotary frequency (``paged.rope_sections``); ``window``: the last queries of a prompt that
    its slots' weights come from, where the cache evicts."""

    def __init__(self, shape: ModelShape, cache, batch: int, max_positions: int, device, dtype=torch.bfloat16, seed: int = 0,
                 std: float = 0.02, layers: int | None = None, axis_of=None, window: int = 32):
        super().__init__(shape, cache, batch, max_positions, device, dtype, seed, std, layers)
        self.axis_of = (0,) * 64 if axis_of is None else tuple(axis_of)
        self.axes, self.window, self._places = max(self.axis_of) + 1, window, {}
        self._released = set()                                  # places that no request runs in
        self.positions = torch.zeros((self.axes, batch), dtype=torch.int64, device=device)       # of the next token
        self._next_position = [0] * batch                       # the largest of them, on the host

    def _layer(self, ldx, residual, x, positions, q, attend, keys=None, values=None):
        """One layer over the step's rows; ``attend()`` is called with queries, keys and values in place."""
        s, L = self.shape, self.layers[ldx]
        normed = torch.empty_like(residual)
        rmsnorm(residual if x is None else x, L["norm1"], s.rms_eps, normed, residual=None if x is None else residual)
        self.cache.append(ldx, F.linear(normed, L["wqkv"]), self.cos_sin, positions, self.axis_of, q, keys, values)
        o = F.linear(attend().view(residual.shape[0], -1), L["wo"])
        rmsnorm(o, L["norm2"], s.rms_eps, normed, residual=residual)
        gated = torch.empty((residual.shape[0], s.intermediate), dtype=self.dtype, device=self.device)
        silu_and_mul(F.linear(normed, L["gate_up"]), gated)
        return F.linear(gated, L["down"])

    def _logits(self, residual, x, at=None):
        """``at``: the requests that the rows are of, where they are not all."""
        normed = torch.empty_like(residual)
        rmsnorm(x, self.final_norm, self.shape.rms_eps, normed, residual=residual)
        logits = F.linear(normed, self.lm_head).float()
        if at is None:
            torch.argmax(logits, dim=-1, out=self.next_ids)
        else:
            self.next_ids.index_copy_(0, at, logits.argmax(-1))
        self.input_ids.copy_(self.next_ids)
        return logits

    def _at(self, requests):
        """Their numbers on the device."""
        if requests not in self._places:
            self._places = {requests: self.cache._to_device(requests).long()}
        return self._places[requests]

    def release(self, request: int) -> None:
        """The request is done: its pages go back, and its place may take another prompt."""
        self.cache.release(request)
        self._released.add(request)

    def prefill_forward(self, prompts, positions=None, requests=None) -> torch.Tensor:
        """``prompts``: a tensor of token ids for every request, or for each of ``requests`` (ascending; the others run on);
        ``positions``: ``[axes, tokens]`` for each, from 0 to ``max_positions - 1`` (default: counted up on every axis; given ones are
        looked at, which waits for them).  Logits ``[prompts, vocab]`` of the last tokens; the cache is brought down to its ``keep``
        slots."""
        from .attn_hub import retroinfer_prefill_attn

        s, counts = self.shape, [int(p.numel()) for p in prompts]
        places = tuple(range(self.batch)) if requests is None else tuple(int(b) for b in requests)
        if len(places) != len(counts) or not places or list(places) != sorted(set(places) & set(range(self.batch))):
            raise ValueError(f"expected a prompt for each of the requests, which ascend from 0 to {self.batch - 1}")
        if min(counts) < 1 or any(self.cache.length_of[b] for b in places):
            raise ValueError("expected prompts of a token or more, and their places in the cache empty")
        all_of_them = len(places) == self.batch
        at, each = None if all_of_them else self._at(places), [0] * self.batch
        for b, n in zip(places, counts):
            each[b] = n
        if positions is None:
            ends, least = counts, 0
            positions = [torch.arange(n, device=self.device).expand(self.axes, n) for n in counts]
        else:
            if len(positions) != len(counts) or any(p.dim() != 2 or p.shape[0] < self.axes or p.shape[1] != n for p, n in zip(positions, counts)):
                raise ValueError(f"expected positions [{self.axes}, tokens] for every prompt")
            ends = [n + 1 for n in torch.stack([p.max() for p in positions]).tolist()]
            least = torch.stack([p.min() for p in positions]).min().item()
        if least < 0 or max(ends) > self.cos_sin.shape[0]:
            raise ValueError(f"positions {least} to {max(ends) - 1}: the table has 0 to {self.cos_sin.shape[0] - 1}")
        where = torch.cat(list(positions), 1).to(torch.int64).contiguous()
        after = self.cache._to_device(ends).long().expand(self.axes, -1)
        rows = sum(counts)
        starts = [sum(counts[:i]) for i in range(len(counts))]
        new = lambda heads: torch.empty((rows, heads, s.head_dim), dtype=self.dtype, device=self.device)  # noqa: E731
        q, k, v = new(s.q_heads), new(s.kv_heads), new(s.kv_heads)
        residual = self.embed[torch.cat(list(prompts)).to(self.device)]
        recent = torch.zeros((len(places), self.window, s.q_heads, s.head_dim), dtype=self.dtype, device=self.device)
        self.cache.begin(each)
        self._released.difference_update(places)
        for b, end in zip(places, ends):
            self._next_position[b] = end
        if at is None:
            self.positions.copy_(after)
        else:
            self.positions.index_copy_(1, at, after.contiguous())
        x = None
        for ldx in range(self.n_layers):
            def attend():
                return torch.cat([retroinfer_prefill_attn(*(t[None, i:i + n] for t in (q, k, v)), True)[0]
                                  for i, n in zip(starts, counts)])
            x = self._layer(ldx, residual, x, where, q, attend, k, v)
            if self.cache.keep is not None:
                for b, (i, n) in enumerate(zip(starts, counts)):
                    w = min(n, self.window)
                    recent[b, self.window - w:] = q[i + n - w:i + n]
                self.cache.observe(recent, ldx, None if all_of_them else places)
        self.cache.evict(slack=0)
        last = torch.tensor([i + n - 1 for i, n in zip(starts, counts)], device=self.device)
        return self._logits(residual[last], x[last], at)

    def decode_forward(self) -> torch.Tensor:
        """One token of every request that was not released: logits ``[running, vocab]``, the greedy next ids become their
        ``input_ids``."""
        running = tuple(b for b in range(self.batch) if b not in self._released)
        if not running:
            raise ValueError("no request is running")
        # eviction bounds the slots, not the positions: behind the table's end every token would turn by the same angles
        past = [b for b in running if self._next_position[b] >= self.cos_sin.shape[0]]
        if past:
            raise RuntimeError(f"requests {past} are at the end of the {self.cos_sin.shape[0]} positions that the model was made for")
        if len(running) < self.batch:
            return self._decode_some(running)
        torch.index_select(self.embed, 0, self.input_ids, out=self.residual)
        self._step(running, 1)
        x, q = None, self.q.view(self.batch, self.shape.q_heads, self.shape.head_dim)
        for ldx in range(self.n_layers):
            x = self._layer(ldx, self.residual, x, self.positions, q, lambda: self.cache.attend(self.q, ldx, out=self.attn))
        self.cache.evict()
        self.positions.add_(1)
        return self._logits(self.residual, x)

    def _step(self, running, counts) -> None:
        self.cache.begin(counts)
        for b in running:
            self._next_position[b] += 1

    def _decode_some(self, running) -> torch.Tensor:
        at, s = self._at(running), self.shape
        residual, positions = self.embed[self.input_ids[at]], self.positions[:, at]
        q = torch.empty((len(running), 1, s.q_heads, s.head_dim), dtype=self.dtype, device=self.device)
        self._step(running, [int(b in running) for b in range(self.batch)])
        x = None
        for ldx in range(self.n_layers):
            x = self._layer(ldx, residual, x, positions, q.view(len(running), s.q_heads, s.head_dim),
                            lambda: self.cache.attend(q, ldx, requests=running))
        self.cache.evict()
        self.positions.index_add_(1, at, torch.ones_like(positions))
        return self._logits(residual, x, at)
