"""KV cache that hands out its rows page by page and can forget the ones that attention has no use for.

Where ``flash_attn_cache`` reserves ``max_length`` rows for every request, this one shares a pool of pages between them, so what a
batch needs is the sum of its lengths; with ``keep`` every request is held to that many slots by evicting those of least
accumulated attention weight (``paged.paged_evict``), and the pages behind go back to the pool.  One decode step of a model:

    cache.begin(1)                                          # pages and lengths for one more token of every request
    for layer in range(layers):
        cache.append(layer, qkv, cos_sin, positions, axis_of, q)
        out = paged_decode_attn(q, None, None, layer, cache)
    cache.evict()                                           # does nothing until a request is `slack` slots over `keep`, or room ends

and of a prompt: ``begin`` with every request's tokens, ``append`` with ``keys`` and ``values`` for ``retroinfer_prefill_attn``, then
``observe`` with the last queries and ``evict(slack=0)``.  A prompt that takes a released place beside running requests names itself:
``begin([0, 57, 0])``, ``append`` with its rows, ``observe(queries, layer, requests=[1])``; so do decode steps of some requests.
Lengths and pages are known on the host without asking the GPU, so nothing synchronises.
"""
from __future__ import annotations

import torch

from .. import paged
from .cache import KV_Cache


class paged_cache(KV_Cache):
    def __init__(self, layer_num: int, batch_size: int, max_length: int, num_key_value_heads: int, num_heads: int,
                 head_dim: int, dtype: torch.dtype, layer_mapping: dict, num_gpus: int, model_size: int, page_size: int = 16,
                 num_pages: int | None = None, keep: int | None = None, sink: int = 4, recent: int = 64, slack: int = 64) -> None:
        # whatever a later call would refuse, before a prompt has run
        if head_dim != paged.DIM:
            raise ValueError("the paged kernels are built for head_dim 128")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"the paged kernels are built for bfloat16 and float16, not {dtype}")
        if num_key_value_heads < 1 or num_heads % num_key_value_heads or not 1 <= num_heads // num_key_value_heads <= paged.MAX_GROUP:
            raise ValueError(f"{num_heads} query heads over {num_key_value_heads} KV heads: decode takes 1 to {paged.MAX_GROUP} to a KV head")
        if page_size & (page_size - 1) or not 8 <= page_size <= 1024:
            raise ValueError(f"page_size={page_size} is not a power of two from 8 to 1024")
        if min(layer_num, batch_size, max_length) < 1 or (num_pages is not None and num_pages < 1):
            raise ValueError("expected a layer, a request, a slot and a page or more")
        devices = {torch.device(layer_mapping[str(ldx)]) for ldx in range(layer_num)}
        if len(devices) != 1:
            raise ValueError("the layers of a paged cache lie on one GPU (several GPUs share a model by its heads)")
        if keep is not None and (min(sink, recent, slack) < 0 or keep < 1 or sink + recent > keep):
            raise ValueError(f"keep={keep} slots for {sink} first and {recent} last tokens, slack={slack}")
        super().__init__(layer_num, batch_size, max_length, num_key_value_heads, num_heads, head_dim, dtype, layer_mapping,
                         num_gpus, model_size)
        self.device = devices.pop()
        self.page_size, self.keep, self.sink, self.recent, self.slack = page_size, keep, sink, recent, slack
        width = -(-max_length // page_size)                     # pages of the longest request
        self.num_pages = batch_size * width if num_pages is None else num_pages
        shape = (self.num_pages, num_key_value_heads, page_size)
        zeros = lambda *s, kind=dtype: torch.zeros(s, dtype=kind, device=self.device)  # noqa: E731
        self.key_pages = [zeros(*shape, head_dim) for _ in range(layer_num)]
        self.value_pages = [zeros(*shape, head_dim) for _ in range(layer_num)]
        # without eviction nothing asks for weights and token numbers
        self.weight = [zeros(*shape, kind=torch.float32) if keep is not None else None for _ in range(layer_num)]
        self.token = [zeros(*shape, kind=torch.int32) if keep is not None else None for _ in range(layer_num)]
        self.page_table = zeros(batch_size, width, kind=torch.int32)
        # slots in use and tokens so far in front of the step's rows, and with them
        self.held, self.lengths = (zeros(batch_size, kind=torch.int32) for _ in range(2))
        self.seen, self.seen_after = (zeros(batch_size, kind=torch.int32) for _ in range(2))
        self.row_start = None                                   # of the step's rows; None: one row of every request
        self.length_of = [0] * batch_size                       # `lengths` on the host
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._pages = [[] for _ in range(batch_size)]
        self._evicted = [False] * batch_size                    # whose slots are no longer in the order of their tokens
        self._fed = [0] * batch_size                            # tokens of the step
        self._weighed, self._weighing = set(), set()            # requests whose slots were given weights before this step, in it
        self._chosen = {}                                       # the step's tables and lengths, of all and of some requests

    def _to_device(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).pin_memory().to(self.device, non_blocking=True)

    def begin(self, counts) -> None:
        """Room for ``counts`` more tokens of the requests (a number for all, or one each)."""
        same = isinstance(counts, int)
        each = [counts] * self.batch_size if same else [int(n) for n in counts]
        if len(each) != self.batch_size or min(each) < 0:
            raise ValueError("expected a number of tokens for every request")
        wanted = [-(-(n + more) // self.page_size) for n, more in zip(self.length_of, each)]
        if max(n + more for n, more in zip(self.length_of, each)) > self.max_length:
            raise RuntimeError(f"a request of more than max_length {self.max_length} slots")
        fresh = [max(0, w - len(p)) for w, p in zip(wanted, self._pages)]
        if sum(fresh) > len(self._free):
            raise RuntimeError(f"the pool has {len(self._free)} pages left and the step needs {sum(fresh)}")
        where, what = [], []
        for b, n in enumerate(fresh):
            for _ in range(n):
                where.append(b * self.page_table.shape[1] + len(self._pages[b]))
                what.append(self._free.pop())
                self._pages[b].append(what[-1])
        if where:
            both = self._to_device([where, what])
            self.page_table.view(-1).index_copy_(0, both[0].long(), both[1])
        self.length_of = [n + more for n, more in zip(self.length_of, each)]
        self._fed, self._chosen = each, {}
        self._weighed |= self._weighing
        self._weighing = set()
        self.held.copy_(self.lengths)
        self.seen.copy_(self.seen_after)
        if same:
            self.lengths.add_(counts)
            self.seen_after.add_(counts)
        else:
            more = self._to_device(each)
            self.lengths.add_(more)
            self.seen_after.add_(more)
        if same and counts == 1:
            self.row_start = None
        else:
            starts = [0]
            for n in each:
                starts.append(starts[-1] + n)
            self.row_start = self._to_device(starts)
        self.context += max(each)

    def append(self, layer_idx, qkv, cos_sin, positions, axis_of, q, keys=None, values=None) -> None:
        """The step's rows of a layer: rotate, split, and write to the pages (``paged.rope_paged_append``)."""
        paged.rope_paged_append(qkv, cos_sin, positions, axis_of, q, self.key_pages[layer_idx], self.value_pages[layer_idx],
                                self.page_table, self.held, self.row_start, weight=self.weight[layer_idx],
                                token=self.token[layer_idx], seen=self.seen, keys=keys, values=values)

    def _of(self, requests):
        """Page table and lengths, of all requests or of some; the layers of a step share them.  A captured call is replayed in later
        steps, whose requests may be longer: it takes the whole table."""
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            if requests is not None:
                raise RuntimeError("calls over some of the requests cannot be captured: which ones is known on the host")
            return self.page_table, self.lengths
        key = None if requests is None else tuple(int(b) for b in requests)
        if key not in self._chosen:
            # no more columns than the longest request has pages: workspaces and the choice of kernels go by them
            table = self.page_table[:, :max(1, max(len(p) for p in self._pages))]
            if key is None:
                self._chosen[key] = table, self.lengths
                return self._chosen[key]
            if not key or len(set(key)) < len(key) or min(key) < 0 or max(key) >= self.batch_size:
                raise ValueError(f"{key} are not different requests of 0 to {self.batch_size - 1}")
            at = self._to_device(key).long()
            self._chosen[key] = table[at], self.lengths[at]
        return self._chosen[key]

    def attend(self, query_states, layer_idx, out=None, lse=None, requests=None) -> torch.Tensor:
        """Attention of one new token of every request, ``[batch, 1, heads, 128]``, over its slots (``paged.paged_decode``); with
        ``keep`` the slots' weights grow by what they are given.  ``requests``: of these alone, in the order of their queries."""
        table, lengths = self._of(requests)
        if self.keep is not None:
            self._weighing.update(range(self.batch_size) if requests is None else map(int, requests))
        return paged.paged_decode(query_states, self.key_pages[layer_idx], self.value_pages[layer_idx], table, lengths, out=out, lse=lse,
                                  weight=self.weight[layer_idx])

    def observe(self, query_states, layer_idx, requests=None) -> None:
        """Weights from the last queries ``[batch, window, heads, 128]`` of the step's prompts (``paged.paged_observe``).  ``requests``:
        of these alone, in the order of their queries; without it, requests without tokens in the step may not have been observed or
        attended before.  A request that was evicted from cannot be observed: its slots are not in the order of its tokens."""
        if self.keep is None:
            return
        table, lengths = self._of(requests)
        which = range(self.batch_size) if requests is None else [int(b) for b in requests]
        for b in which:
            if self._evicted[b]:
                raise RuntimeError(f"slots of request {b} were evicted: what its queries see is not known any more")
            if requests is None and not self._fed[b] and b in self._weighed and self.length_of[b]:
                raise ValueError(f"request {b} had no tokens in this step: name the `requests` that are to be observed")
        self._weighing.update(which)
        paged.paged_observe(query_states, self.key_pages[layer_idx], table, lengths, self.weight[layer_idx])

    def evict(self, slack: int | None = None) -> bool:
        """Once a request is ``slack`` slots over ``keep``, or over ``keep`` at all where another token of every request would not fit
        ``max_length`` or the pool, bring every request down to ``keep`` and give the pages behind back."""
        over = self.slack if slack is None else slack
        most = max(self.length_of)
        if self.keep is None or most <= self.keep or (most <= self.keep + over and self._room_for_a_token()):
            return False
        table, lengths = self._of(None)
        for ldx in range(self.layer_num):
            paged.paged_evict(self.key_pages[ldx], self.value_pages[ldx], self.weight[ldx], self.token[ldx], table, lengths, self.seen_after,
                              self.keep, self.sink, self.recent)
        self.lengths.clamp_(max=self.keep)
        self._evicted = [e or n > self.keep for e, n in zip(self._evicted, self.length_of)]
        self._chosen = {}
        self.length_of = [min(n, self.keep) for n in self.length_of]
        for b, n in enumerate(self.length_of):
            self._give_back(b, -(-n // self.page_size))
        return True

    def _room_for_a_token(self) -> bool:
        """Of every request."""
        fresh = sum(n + 1 > len(p) * self.page_size for n, p in zip(self.length_of, self._pages))
        return max(self.length_of) < self.max_length and fresh <= len(self._free)

    def release(self, bdx: int) -> None:
        """Request ``bdx`` is done: its pages go back, and its place may take another one."""
        self._give_back(bdx, 0)
        self.length_of[bdx], self._evicted[bdx], self._fed[bdx], self._chosen = 0, False, 0, {}
        self._weighed.discard(bdx)
        self._weighing.discard(bdx)
        for x in (self.lengths, self.seen_after):
            x[bdx].zero_()

    def _give_back(self, bdx: int, keep_pages: int) -> None:
        self._free.extend(reversed(self._pages[bdx][keep_pages:]))
        del self._pages[bdx][keep_pages:]

    @property
    def free_pages(self) -> int:
        return len(self._free)
