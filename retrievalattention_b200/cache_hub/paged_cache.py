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

Layers may look back over a window (``attn_window``, ``attn_sink``): ``attend`` and ``prompt`` go by it.  ``prompt`` is the attention of
the step's rows over the pages, for prompts that follow on what is cached.  ``share(0, [1, 2])``: empty requests begin with the pages of
request 0, whose prompt has run, and ``attend`` reads what they have in common once for all of them, where that is enough to be faster.
"""
from __future__ import annotations

import torch

from .. import paged
from .cache import KV_Cache


class paged_cache(KV_Cache):
    def __init__(self, layer_num: int, batch_size: int, max_length: int, num_key_value_heads: int, num_heads: int,
                 head_dim: int, dtype: torch.dtype, layer_mapping: dict, num_gpus: int, model_size: int, page_size: int = 16,
                 num_pages: int | None = None, keep: int | None = None, sink: int = 4, recent: int = 64, slack: int = 64,
                 attn_window=None, attn_sink: int = 0) -> None:
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
        windows = list(attn_window) if isinstance(attn_window, (list, tuple)) else [attn_window] * layer_num
        if len(windows) != layer_num or any(w is not None and (w != int(w) or w < 1) for w in windows) or attn_sink != int(attn_sink) or attn_sink < 0:
            raise ValueError(f"attn_window={attn_window}, attn_sink={attn_sink}: expected a slot or more (or None) for all layers or each")
        if keep is not None and any(w is not None for w in windows):
            raise ValueError("a window goes by the order of the slots, which eviction does not keep: attn_window or keep")
        super().__init__(layer_num, batch_size, max_length, num_key_value_heads, num_heads, head_dim, dtype, layer_mapping,
                         num_gpus, model_size)
        self.device = devices.pop()
        self.attn_window, self.attn_sink = [None if w is None else int(w) for w in windows], int(attn_sink)
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
        # of the step's rows, in one place, so that captured calls follow it; row_start None: one row of every request
        self._one_each = torch.arange(batch_size + 1, dtype=torch.int32, device=self.device)
        self._row_start, self.row_start = self._one_each.clone(), None
        self.length_of = [0] * batch_size                       # `lengths` on the host
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._pages = [[] for _ in range(batch_size)]
        self._evicted = [False] * batch_size                    # whose slots are no longer in the order of their tokens
        self._fed = [0] * batch_size                            # tokens of the step
        self._weighed, self._weighing = set(), set()            # requests whose slots were given weights before this step, in it
        self._chosen = {}                                       # the step's tables and lengths, of all and of some requests
        self._sharers = {}                                      # page: requests that begin with it, where they are several
        # group_start and shared of `paged.paged_shared_decode`, as many groups as requests, so that captured calls follow them
        self._group_start, self._group_shared = zeros(batch_size + 1, kind=torch.int32), zeros(batch_size, kind=torch.int32)
        self._alike, self._together = False, False              # some next to each other have slots in common, and enough of them
        self._grouped = {}                                      # groups of some of the requests

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
            if self.row_start is not None:
                self._row_start.copy_(self._one_each)
            self.row_start = None
        else:
            starts = [0]
            for n in each:
                starts.append(starts[-1] + n)
            self._row_start.copy_(self._to_device(starts))
            self.row_start = self._row_start
        self.context += max(each)

    def append(self, layer_idx, qkv, cos_sin, positions, axis_of, q, keys=None, values=None, q_norm=None, k_norm=None, eps=1e-6) -> None:
        """The step's rows of a layer: normalise heads where weights are given, rotate, split, and write to the pages
        (``paged.rope_paged_append``).  A captured call goes by the rows that later steps' ``begin`` shares out."""
        paged.rope_paged_append(qkv, cos_sin, positions, axis_of, q, self.key_pages[layer_idx], self.value_pages[layer_idx],
                                self.page_table, self.held, self._row_start if self._captures() else self.row_start, weight=self.weight[layer_idx],
                                token=self.token[layer_idx], seen=self.seen, keys=keys, values=values, q_norm=q_norm, k_norm=k_norm,
                                eps=eps)

    def _captures(self) -> bool:
        return self.device.type == "cuda" and torch.cuda.is_current_stream_capturing()

    def _of(self, requests):
        """Page table and lengths, of all requests or of some; the layers of a step share them.  A captured call is replayed in later
        steps, whose requests may be longer: it takes the whole table."""
        if self._captures():
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
        """Attention of one new token of every request, ``[batch, 1, heads, 128]``, over its slots (``paged.paged_decode``), or the
        layer's window of them; with ``keep`` the slots' weights grow by what they are given.  ``requests``: of these alone, in the order of
        their queries.  Slots that requests next to each other, in that order, have in common are read once (``paged.paged_shared_decode``),
        where they are many enough."""
        table, lengths = self._of(requests)
        pools, window = (self.key_pages[layer_idx], self.value_pages[layer_idx]), self.attn_window[layer_idx]
        if window is not None:
            return paged.paged_decode(query_states, *pools, table, lengths, out=out, lse=lse, window=window, sink=self.attn_sink)
        groups = self._groups_of(requests)
        if groups is not None:
            return paged.paged_shared_decode(query_states, *pools, table, lengths, *groups, out=out, lse=lse)
        if self.keep is not None:
            self._weighing.update(range(self.batch_size) if requests is None else map(int, requests))
        return paged.paged_decode(query_states, *pools, table, lengths, out=out, lse=lse, weight=self.weight[layer_idx])

    def prompt(self, query_states, layer_idx, out=None, lse=None) -> torch.Tensor:
        """Attention of the step's rows ``[rows, heads, 128]``, as ``append`` had them, over their requests' slots, or the layer's window
        of them (``paged.paged_prompt``).  Not of a request that was evicted from."""
        if any(e and n for e, n in zip(self._evicted, self._fed)):
            raise RuntimeError("slots of a request were evicted: what its rows see is not known any more")
        table, lengths = self._of(None)
        return paged.paged_prompt(query_states, self.key_pages[layer_idx], self.value_pages[layer_idx], table, lengths, self._row_start,
                                  window=self.attn_window[layer_idx], sink=self.attn_sink, out=out, lse=lse)

    def share(self, of: int, requests, slots: int | None = None) -> int:
        """Let ``requests``, which are empty, begin with the first ``slots`` slots of request ``of`` (default: all of them), as far as
        they fill pages: nothing is copied.  Returns how many they are.  Not with ``keep``: requests that share pages cannot be evicted
        from."""
        if not 0 <= of < self.batch_size:
            raise ValueError(f"request {of} of {self.batch_size}")
        requests, n = [int(b) for b in requests], self.length_of[of] if slots is None else slots
        if self.keep is not None:
            raise ValueError("requests that share pages cannot be evicted from: share or keep")
        if not 0 <= n <= self.length_of[of] or of in requests or len(set(requests)) < len(requests) or \
                any(not 0 <= b < self.batch_size or self.length_of[b] for b in requests):
            raise ValueError(f"expected up to {self.length_of[of]} slots and empty requests other than {of}")
        pages = self._pages[of][:n // self.page_size]
        n = len(pages) * self.page_size
        if not pages or not requests:
            return n
        for id in pages:
            self._sharers[id] = self._sharers.get(id, 1) + len(requests)
        at = self._to_device(requests).long()
        self.page_table[at, :len(pages)] = self._to_device(pages)
        for x in (self.lengths, self.seen_after):
            x.index_fill_(0, at, n)
        for b in requests:
            self._give_back(b, 0)
            self._pages[b], self.length_of[b] = list(pages), n
        self._chosen = {}
        self._regroup()
        return n

    def _in_common(self, which):
        """Runs of requests next to each other in ``which`` that begin with the same pages, so that the fewest slots are read: the first of
        every run (and the end), the slots that it has in common."""
        def alike(a, b):                                        # by halves: lists of thousands of pages, between two steps
            low, high = 0, min(len(a), len(b))
            while low < high:
                mid = (low + high + 1) // 2
                low, high = (mid, high) if a[low:mid] == b[low:mid] else (low, mid - 1)
            return low

        pages = [self._pages[b] for b in which]
        common = [alike(a, b) for a, b in zip(pages, pages[1:])]
        best = [(0, 0, 0)]                                      # of the first j requests: pages saved, where the last run begins, its pages
        for j in range(1, len(pages) + 1):
            top, least = (best[j - 1][0], j - 1, 0), None
            for i in range(j - 2, max(-1, j - 513), -1):        # a run of more than 512 may as well be two
                least = common[i] if least is None else min(least, common[i])
                if least == 0:
                    break
                top = max(top, (best[i][0] + (j - 1 - i) * least, i, least))
            best.append(top)
        starts, shared, j = [len(pages)], [], len(pages)
        while j > 0:
            _, j, n = best[j]
            starts.append(j)
            shared.append(n * self.page_size)
        return starts[::-1], shared[::-1]

    # What is read once for several requests has to be this many MB of keys and values less, and as many more for each request, or they
    # are attended one by one: it takes two kernels more, and what others have just read is often found in L2.  8 heads of 4, one by one and
    # together: 2 requests of 65536 slots in common (268 MB) 85 and 87 us, 8 of 8192 (235 MB) 50 and 48, of 16384 (470 MB) 85 and 60, 64 of
    # 2048 (529 MB) 97 and 81, of 1024 in front of 4096 of their own (264 MB) 206 and 247, 256 of 512 (535 MB) 149 and 210, of 2048 351 and 214.
    _PAYS_MB, _PAYS_MB_EACH = 256, 4

    def _pays(self, starts, shared) -> bool:
        saved = sum((j - i - 1) * n for i, j, n in zip(starts, starts[1:], shared))
        return saved > 0 and saved * self.kv_head * 4 * paged.DIM >= (self._PAYS_MB + self._PAYS_MB_EACH * starts[-1]) << 20

    def _groups_of(self, requests):
        """Of all requests, or of some in their order; None where one by one is faster.  Captured calls take what is alike now for a sign
        of what later steps have in common."""
        if requests is None:
            return (self._group_start, self._group_shared) if self._alike and (self._together or self._captures()) else None
        if not self._sharers:
            return None
        key = tuple(int(b) for b in requests)
        if key not in self._grouped:
            starts, shared = self._in_common(key)
            if len(self._grouped) > 15:                         # kept over the steps, not for every choice that there ever was
                self._grouped = {}
            self._grouped[key] = (self._to_device(starts), self._to_device(shared)) if self._pays(starts, shared) else None
        return self._grouped[key]

    def _regroup(self) -> None:
        self._grouped = {}
        starts, shared = self._in_common(range(self.batch_size))
        more = self.batch_size - len(shared)
        self._group_start.copy_(self._to_device(starts + [self.batch_size] * more))
        self._group_shared.copy_(self._to_device(shared + [0] * more))
        self._alike, self._together = any(shared), self._pays(starts, shared)

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
        if self._alike or self._grouped:
            self._regroup()
        self._weighed.discard(bdx)
        self._weighing.discard(bdx)
        for x in (self.lengths, self.seen_after):
            x[bdx].zero_()

    def _give_back(self, bdx: int, keep_pages: int) -> None:
        for id in reversed(self._pages[bdx][keep_pages:]):
            left = self._sharers.get(id, 1) - 1
            if left == 0:
                self._free.append(id)
            if left > 1:
                self._sharers[id] = left
            else:
                self._sharers.pop(id, None)
        del self._pages[bdx][keep_pages:]

    @property
    def free_pages(self) -> int:
        return len(self._free)
