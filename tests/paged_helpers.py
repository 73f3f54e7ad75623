"""A paged cache for tests, and the operators' definitions in 64 bits on the CPU."""
import math

import torch

DIM = 128


class Layer:
    """One layer of a paged cache on the GPU: requests of `lengths` slots on shuffled pages.  What no request uses is NaN in the
    pools and -1 in the page table.  `apart`: pages of keys and of values interleaved in one tensor."""

    def __init__(self, lengths, kv_heads, page, dtype, seed=0, room=0, spare=2, apart=False, first_page=0):
        gen = torch.Generator().manual_seed(seed)
        self.lengths_list, self.hk, self.page, self.dtype = list(lengths), kv_heads, page, dtype
        used = [-(-(n + room) // page) for n in lengths]
        n_pages = first_page + sum(used) + spare
        order = (torch.randperm(n_pages - first_page, generator=gen) + first_page).tolist()
        self.pages_of = []
        for n in used:
            self.pages_of.append(order[:n])
            order = order[n:]
        width = max(1, max(used) + 1)
        table = torch.full((len(used), width), -1, dtype=torch.int32)
        for b, ids in enumerate(self.pages_of):
            table[b, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        self.table = table.cuda()
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.gen = gen
        shape = (n_pages, kv_heads, page, DIM)
        if apart:
            both = torch.full((n_pages, 2, kv_heads, page, DIM), float("nan"), dtype=dtype, device="cuda")
            self.keys, self.values = both[:, 0], both[:, 1]
        elif first_page:
            self.keys, self.values = torch.empty(shape, dtype=dtype, device="cuda"), torch.empty(shape, dtype=dtype, device="cuda")
        else:
            self.keys, self.values = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        self.weight = torch.full(shape[:3], float("nan"), device="cuda")
        self.token = torch.full(shape[:3], -7, dtype=torch.int32, device="cuda")
        self.k, self.v, self.w, self.t = [], [], [], []          # per request: [kv_heads, slots(, 128)] in 64 bits
        for b, n in enumerate(lengths):
            k, v = (torch.randn((kv_heads, n, DIM), generator=gen).to(dtype) for _ in range(2))
            w = torch.rand((kv_heads, n), generator=gen)
            t = torch.arange(n, dtype=torch.int32).expand(kv_heads, n).contiguous()
            self.fill(b, k, v, w, t)

    def fill(self, b, k, v, w, t):
        """Request b's slots: [kv_heads, slots(, 128)]."""
        while len(self.k) <= b:
            for x in (self.k, self.v, self.w, self.t):
                x.append(None)
        self.k[b], self.v[b], self.w[b], self.t[b] = k.double(), v.double(), w.double(), t.clone()
        self.scatter(self.keys, b, k)
        self.scatter(self.values, b, v)
        self.scatter(self.weight, b, w)
        self.scatter(self.token, b, t)

    def scatter(self, pool, b, x):
        for i, id in enumerate(self.pages_of[b]):
            part = x[:, i * self.page:(i + 1) * self.page]
            if part.shape[1]:
                pool[id, :, :part.shape[1]] = part.to(pool.device)

    def gather(self, pool, b, n=None):
        """Request b's slots of a pool, on the CPU: [kv_heads, slots(, 128)]."""
        n = self.lengths_list[b] if n is None else n
        if n == 0:
            return pool[:0, 0].cpu().reshape(self.hk, 0, *pool.shape[3:])
        x = pool[torch.tensor(self.pages_of[b], device=pool.device)].transpose(0, 1)
        return x.reshape(self.hk, -1, *pool.shape[3:])[:, :n].cpu()


def attend(q, k, v, allowed=None, scale=DIM ** -0.5):
    """q [heads, rows, 128] against k, v [heads, slots, 128], all in 64 bits: (out, lse, probabilities)."""
    s = q @ k.transpose(-1, -2) * scale
    if allowed is not None:
        s = s.masked_fill(~allowed, -math.inf)
    lse = torch.logsumexp(s, -1) if k.shape[-2] else torch.full(s.shape[:-1], -math.inf, dtype=torch.float64)
    p = torch.where(torch.isfinite(lse)[..., None], torch.exp(s - lse[..., None]), torch.zeros_like(s))
    return p @ v, lse, p


def rounding(dtype):
    """Half a unit in the last place, relative; and the spacing of the smallest values."""
    return (2.0 ** -8, 2.0 ** -130) if dtype == torch.bfloat16 else (2.0 ** -11, 2.0 ** -25)
