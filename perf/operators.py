"""The operators around a paged KV cache, as measurable cases.

Four operators, all through ``retrievalattention_b200.paged``, on one cache layer: pools of pages ``[pages, kv_heads, page, 128]``
for keys and values, with the accumulated attention weight and the token number of every slot beside them, and a page table and a
length for each request.

* ``append``   ``rope_paged_append``: rotary positions with several axes on a fused QKV projection; queries out, keys and values
               into the pages;
* ``decode``   ``paged_decode``: attention of one new token over the pages, optionally adding its weights to the slots';
* ``observe``  ``paged_observe``: the weights that a prompt's last queries give to its slots;
* ``evict``    ``paged_evict``: the slots of least weight give way, in place.

The plain forms are elementary torch operations in 32 bits.  Page 0 of a pool belongs to no request; page tables are filled up with it.
"""
import math

import torch

own = False

DIM = 128
THETA = 1e6
STALE = 0.25                             # scale of what lies in slots that no request uses
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # -- append.  `tokens` rows of the longest request, `least` of the shortest; `held`: tokens already cached
        # a decode step of four requests: launches count
        dict(name="append-step-b4", kind="append", batch=4, kv_heads=8, group=4, tokens=1, least=1, held=2000, page=16,
             sections="16,24,24", interleaved=False, dtype="bf16"),
        # three prompts with images, of odd lengths, into a cache that holds a system prompt; seven query heads a group
        dict(name="append-ragged-b3", kind="append", batch=3, kv_heads=4, group=7, tokens=5001, least=77, held=333, page=32,
             sections="24,20,20", interleaved=True, dtype="fp16"),
        # one long prompt with video frames
        dict(name="append-32k", kind="append", batch=1, kv_heads=8, group=4, tokens=32768, least=32768, held=0, page=64,
             sections="16,24,24", interleaved=False, dtype="bf16"),
        # -- decode.  `tokens` slots of the longest request, `least` of the shortest
        # one user, a short question: latency
        dict(name="decode-777", kind="decode", batch=1, kv_heads=8, group=4, tokens=777, least=777, page=16, weights=False,
             dtype="bf16"),
        # a serving batch of uneven requests, the newest of them without a slot yet, with weights for eviction
        dict(name="decode-5k-b16-ragged", kind="decode", batch=16, kv_heads=4, group=7, tokens=5003, least=0, page=8,
             weights=True, dtype="fp16"),
        # documents of 20K to 32K tokens, with weights
        dict(name="decode-32k-b4", kind="decode", batch=4, kv_heads=8, group=4, tokens=32768, least=20011, page=64,
             weights=True, dtype="bf16"),
        # Llama-3-8B geometry, 128K context, batch 4: the benchmark's default geometry, every slot attended
        dict(name="decode-128k-b4", kind="decode", batch=4, kv_heads=8, group=4, tokens=131072, least=131072, page=16,
             weights=False, dtype="bf16"),
        # -- observe.  `window`: queries at the prompt's end
        # a short prompt
        dict(name="observe-1k", kind="observe", batch=1, kv_heads=8, group=4, tokens=1001, least=1001, window=16, page=16,
             dtype="bf16"),
        # documents of 20K to 32K tokens, window of 64 queries: 256 rows a KV head
        dict(name="observe-32k-b4", kind="observe", batch=4, kv_heads=8, group=4, tokens=32768, least=20011, window=64, page=64,
             dtype="bf16"),
        # -- evict.  `keep` slots remain, the first `sink` and last `recent` tokens among them
        # a short prompt, half of it
        dict(name="evict-1k", kind="evict", batch=1, kv_heads=8, tokens=1001, least=1001, keep=512, sink=4, recent=64, page=16,
             dtype="bf16"),
        # every 64 generated tokens: requests that hold 64 slots more than they may
        dict(name="evict-step-b16", kind="evict", batch=16, kv_heads=8, tokens=4160, least=4160, keep=4096, sink=4, recent=64,
             page=32, dtype="bf16"),
        # documents of 20K to 32K tokens, down to 8K
        dict(name="evict-32k-b4", kind="evict", batch=4, kv_heads=8, tokens=32768, least=20011, keep=8192, sink=4, recent=64,
             page=64, dtype="fp16"),
    ]


def _between(rng, low, high):
    """A whole number from low to high, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "observe", "evict"))
    kv_heads, group = rng.choice(((8, 4), (4, 7), (1, 8), (2, 8), (8, 8), (4, 1), (2, 5), (8, 2)))
    case = dict(kind=kind, kv_heads=kv_heads, page=rng.choice((8, 16, 16, 32, 64, 128)), dtype=rng.choice(("bf16", "bf16", "fp16")))
    if kind != "evict":
        case["group"] = group
    if kind == "append":
        step = rng.random() < 0.4
        tokens = 1 if step else _between(rng, 2, 30000)
        case["batch"] = _between(rng, 1, 100) if step else rng.randint(1, max(1, min(6, 30000 // tokens)))
        case["held"] = rng.choice((0, _between(rng, 1, 4000)))
        case["sections"], case["interleaved"] = rng.choice((("16,24,24", False), ("24,20,20", True), ("64", False), ("32,32", False)))
        least = 1
    else:
        most = {"decode": 1 << 22, "observe": 1 << 20, "evict": 1 << 20}[kind]      # slots of all requests and KV heads
        tokens = _between(rng, 20, 120000 if kind == "decode" else 30000)
        case["batch"] = _between(rng, 1, max(1, min(64, most // (tokens * kv_heads))))
        least = rng.choice((0, 1))
    case["tokens"] = tokens
    case["least"] = rng.choice((tokens, rng.randint(least, tokens)))
    if kind == "decode":
        case["weights"] = rng.random() < 0.5
    if kind == "observe":
        case["window"] = rng.randint(1, max(1, min(64, 256 // group)))
    if kind == "evict":
        case["keep"] = rng.randint(1, max(1, tokens - 1))
        case["sink"] = min(4, case["keep"] // 4)
        case["recent"] = min(rng.choice((0, 16, 64)), case["keep"] // 2)
    return case


def _spread(case):
    """Tokens of every request: from `tokens` (first request) to `least` (last one)."""
    b = case["batch"]
    return [case["tokens"]] if b == 1 else [case["tokens"] - (case["tokens"] - case["least"]) * i // (b - 1) for i in range(b)]


def _axis_of(case):
    """The axis that each of the 64 frequencies follows: one section behind the other, or dealt out in turn while they last."""
    left = [int(n) for n in case["sections"].split(",")]
    if not case["interleaved"]:
        return tuple(a for a, n in enumerate(left) for _ in range(n))
    axes, a = [], 0
    while len(axes) < DIM // 2:
        if left[a]:
            left[a] -= 1
            axes.append(a)
        a = (a + 1) % len(left)
    return tuple(axes)


def _image_positions(n, axes):
    """Positions [axes, n] of text with images: 232 tokens of text, then an image of 24 x 32 patches, again and again."""
    i = torch.arange(n, device="cuda")
    base, j = i // 1000 * (232 + 32), i % 1000
    patch = (j - 232).clamp(min=0)
    text = base + j.clamp(max=232)
    inside = j >= 232
    rows = [text, torch.where(inside, base + 232 + patch // 32, text), torch.where(inside, base + 232 + patch % 32, text)]
    return torch.stack(rows[:axes])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 1)
    kind, dtype, b, hk, page = case["kind"], DTYPES[case["dtype"]], case["batch"], case["kv_heads"], case["page"]
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    tokens = _spread(case)
    held = case.get("held", 0)
    used = [-(-(n + held) // page) for n in tokens]                  # pages of every request
    width, pages = max(1, max(used)), 1 + sum(used) + 3
    ids = (torch.randperm(pages - 1, generator=gen, device="cuda") + 1).to(torch.int32)
    table = torch.zeros((b, width), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = ids[at:at + n]
        at += n
    # keys with channels of uneven size, as rotated keys have them
    shape = (pages, hk, page, DIM)
    keys = torch.empty(shape, dtype=dtype, device="cuda")
    values = torch.empty(shape, dtype=dtype, device="cuda")
    size = 0.5 + randn(1, hk, 1, DIM).abs()
    step = max(1, (1 << 27) // (hk * page * DIM))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        keys[p:p + n] = (randn(n, hk, page, DIM) * size).to(dtype)
        values[p:p + n] = randn(n, hk, page, DIM).to(dtype)
    keys[0] *= STALE
    values[0] *= STALE
    state = dict(case=case, keys=keys, values=values, table=table)
    if kind == "append":
        hq, axis_of = hk * case["group"], _axis_of(case)
        axes, rows = max(axis_of) + 1, sum(tokens)
        state["qkv"] = randn(rows, (hq + 2 * hk) * DIM).to(dtype)
        positions = [_image_positions(n, axes) if n > 1 else torch.full((axes, 1), 900 + i, device="cuda") for i, n in enumerate(tokens)]
        state["positions"] = torch.cat(positions, 1).long().contiguous()
        most = held + max(max(tokens), 1000) + 1000
        freq = torch.outer(torch.arange(most, dtype=torch.float32, device="cuda"),
                           1.0 / THETA ** (torch.arange(0, DIM, 2, dtype=torch.float32, device="cuda") / DIM))
        state["cos_sin"] = torch.cat((freq.cos(), freq.sin()), -1).contiguous()
        state["axis_of"] = axis_of
        state["q"] = torch.zeros((rows, hq, DIM), dtype=dtype, device="cuda")
        state["row_start"] = torch.tensor([0] + tokens, device="cuda").cumsum(0).to(torch.int32)
        state["lengths"] = torch.full((b,), held, dtype=torch.int32, device="cuda")
        state["seen"] = state["lengths"] + 7                         # seven tokens were evicted before
        state["weight"] = randn(pages, hk, page).abs()
        state["token"] = torch.zeros((pages, hk, page), dtype=torch.int32, device="cuda")
        return state
    state["lengths"] = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    # slots' weights: a few large, many small, some none at all
    weight = randn(pages, hk, page).exp() * 1e-4
    weight[torch.rand(weight.shape, generator=gen, device="cuda") < 0.05] = 0.0
    if kind == "evict":
        # slots in the order of an earlier eviction: mostly ascending tokens
        slot = torch.arange(width * page, device="cuda")
        token = torch.stack([(slot + 100) * (slot >= 64) + (slot * 3 + 5) * (slot < 64) * (slot >= 4) + slot * (slot < 4)] * hk)
        paged = token.reshape(hk, width, page).transpose(0, 1).to(torch.int32)
        tokens_of = torch.zeros((pages, hk, page), dtype=torch.int32, device="cuda")
        for i, n in enumerate(used):
            tokens_of[table[i, :n].long()] = paged[:n]
        state["before"] = torch.stack((weight.view(torch.int32), tokens_of))      # what the slots' records are before the call
        state["records"] = state["before"].clone()
        state["seen"] = state["lengths"] + 100
        return state
    state["weight"] = weight
    hq, rows = hk * case["group"], case.get("window", 1)
    state["q"] = randn(b, rows, hq, DIM).to(dtype)
    return state


def _of_slots(pool, table):
    """[pages, heads, page, ...] -> [batch, heads, slots, ...], in 32 bits."""
    x = pool[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:]).float()


def _probabilities(q, k, seen):
    """Softmax over the slots that `seen` allows, and its log-sum-exp; rows that see none are zero."""
    s = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(DIM)
    s = torch.where(seen, s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(m), m, 0.0))
    total = e.sum(-1, keepdim=True)
    lse = torch.where(total > 0, m + torch.log(total), float("-inf"))[..., 0]
    return e / torch.where(total > 0, total, 1.0), lse


def _add_weights(pool, table, add):
    """add [batch, heads, slots] to the slots' weights."""
    b, h, n = add.shape
    page = pool.shape[2]
    pool.index_add_(0, table.reshape(-1).long(), add.reshape(b, h, n // page, page).transpose(1, 2).reshape(-1, h, page))


def _plain_append(s):
    qkv, table, keys, values = s["qkv"], s["table"], s["keys"], s["values"]
    rows, hq, hk, page = qkv.shape[0], s["q"].shape[1], keys.shape[1], keys.shape[2]
    axis_of = torch.tensor(s["axis_of"], device="cuda")
    angle = s["cos_sin"][s["positions"]]                              # [axes, rows, 128]
    i = torch.arange(DIM // 2, device="cuda")
    cos, sin = angle[axis_of, :, i].t()[:, None], angle[axis_of, :, DIM // 2 + i].t()[:, None]
    x = qkv.view(rows, hq + 2 * hk, DIM)
    turned = x[:, :hq + hk].float()
    a, b = turned[..., :DIM // 2], turned[..., DIM // 2:]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(qkv.dtype)
    s["q"].copy_(turned[:, :hq])
    row = torch.arange(rows, device="cuda")
    request = torch.searchsorted(s["row_start"].long(), row, right=True) - 1
    place = row - s["row_start"].long()[request]
    slot = s["lengths"].long()[request] + place
    at = table.long()[request, slot // page]
    keys[at, :, slot % page] = turned[:, hq:]
    values[at, :, slot % page] = x[:, hq + hk:]
    s["weight"][at, :, slot % page] = 0.0
    s["token"][at, :, slot % page] = (s["seen"].long()[request] + place).to(torch.int32)[:, None]
    return {"q": s["q"], "keys": keys, "values": values, "weight": s["weight"], "token": s["token"]}


def _plain_decode(s):
    case, q = s["case"], s["q"]
    b, _, hq, d = q.shape
    hk = s["keys"].shape[1]
    k, v = _of_slots(s["keys"], s["table"]), _of_slots(s["values"], s["table"])
    seen = torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None, None, None]
    p, lse = _probabilities(q.view(b, hk, hq // hk, d).float(), k, seen)
    out = {"out": torch.matmul(p, v).reshape(b, 1, hq, d).to(q.dtype), "lse": lse.reshape(b, hq)}
    if case["weights"]:
        _add_weights(s["weight"], s["table"], p.sum(2))
        out["weight"] = s["weight"]
    return out


def _plain_observe(s):
    q = s["q"]
    b, w, hq, d = q.shape
    hk = s["keys"].shape[1]
    k = _of_slots(s["keys"], s["table"])
    slot = torch.arange(k.shape[2], device="cuda")
    last = s["lengths"][:, None] - w + torch.arange(w, device="cuda")                 # slot of a query's own token
    seen = (slot <= last[..., None])[:, None, :, None].expand(b, 1, w, hq // hk, -1).reshape(b, 1, w * (hq // hk), -1)
    rows = q.view(b, w, hk, hq // hk, d).transpose(1, 2).reshape(b, hk, -1, d).float()
    p, _ = _probabilities(rows, k, seen)
    _add_weights(s["weight"], s["table"], p.sum(2))
    return s["weight"]


def _plain_evict(s, records):
    case, table, lengths = s["case"], s["table"].long(), s["lengths"].long()
    keep, page, hk = case["keep"], case["page"], case["kv_heads"]
    b, n = table.shape[0], table.shape[1] * page
    slot = torch.arange(n, device="cuda")
    weight, token = (x[table].transpose(1, 2).reshape(b, hk, n) for x in (records[0].view(torch.float32), records[1]))
    protected = (token < case["sink"]) | (token >= s["seen"][:, None, None] - case["recent"])
    rank = torch.where(protected, float("inf"), weight)
    rank = torch.where(slot < lengths[:, None, None], rank, float("-inf"))
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :keep]
    kept = torch.zeros((b, hk, n), dtype=torch.bool, device="cuda").scatter_(-1, order, True) & (slot < lengths[:, None, None])
    behind = kept & (slot >= keep)                                                    # these move into the holes in front
    hole = ~kept & (slot < torch.clamp(lengths, max=keep)[:, None, None])
    room = n + 1
    source = torch.zeros((b, hk, room), dtype=torch.long, device="cuda")
    source.scatter_(-1, torch.where(behind, behind.cumsum(-1) - 1, n), slot.expand(b, hk, n))
    taken = torch.where(hole, source.gather(-1, torch.where(hole, hole.cumsum(-1) - 1, n)), slot)[..., :keep]
    head = torch.arange(hk, device="cuda")[None, :, None]
    row = lambda at: (table[torch.arange(b, device="cuda")[:, None, None], at // page] * hk + head) * page + at % page  # noqa: E731
    to, of = row(slot[:keep].expand(b, hk, -1)).reshape(-1), row(taken).reshape(-1)
    for pool in (s["keys"].view(-1, DIM), s["values"].view(-1, DIM), records[0].view(-1), records[1].view(-1)):
        pool[to] = pool[of]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "evict":
        records = s["records"].copy_(s["before"])
        weight, token = records[0].view(torch.float32), records[1]
        out = {"keys": s["keys"], "values": s["values"], "weight": weight, "token": token}
        if own:
            from retrievalattention_b200 import paged
            paged.paged_evict(s["keys"], s["values"], weight, token, s["table"], s["lengths"], s["seen"], case["keep"],
                              case["sink"], case["recent"])
        else:
            _plain_evict(s, records)
        return out
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "observe": _plain_observe}[kind](s)
    from retrievalattention_b200 import paged
    if kind == "append":
        paged.rope_paged_append(s["qkv"], s["cos_sin"], s["positions"], s["axis_of"], s["q"], s["keys"], s["values"], s["table"],
                                s["lengths"], s["row_start"], weight=s["weight"], token=s["token"], seen=s["seen"])
        return {"q": s["q"], "keys": s["keys"], "values": s["values"], "weight": s["weight"], "token": s["token"]}
    if kind == "decode":
        weight = s["weight"] if case["weights"] else None
        lse = torch.empty((case["batch"], s["q"].shape[2]), dtype=torch.float32, device="cuda")
        out = {"out": paged.paged_decode(s["q"], s["keys"], s["values"], s["table"], s["lengths"], lse=lse, weight=weight), "lse": lse}
        if weight is not None:
            out["weight"] = weight
        return out
    paged.paged_observe(s["q"], s["keys"], s["table"], s["lengths"], s["weight"])
    return s["weight"]


def work(case):
    kind, hk, tokens = case["kind"], case["kv_heads"], _spread(case)
    slots = sum(tokens) * hk
    if kind == "append":
        rows, heads = sum(tokens), hk * case["group"] + 2 * hk
        axes = len(case["sections"].split(","))
        # the projection in, queries and cache rows out, a table row and the positions in, weights and token numbers out
        return {"bytes": rows * (2 * heads * DIM * 2 + 4 * DIM + 8 * axes) + 8 * slots, "flops": rows * (heads - hk) * DIM * 3}
    if kind == "decode":
        hq = hk * case["group"]
        return {"bytes": slots * (4 * DIM + (8 if case["weights"] else 0)) + case["batch"] * hq * (4 * DIM + 4),
                "flops": 4 * DIM * sum(tokens) * hq}
    if kind == "observe":
        rows = case["window"] * case["group"]
        return {"bytes": slots * (2 * DIM + 8) + 2 * DIM * rows * hk * case["batch"], "flops": 2 * DIM * rows * slots}
    # evict: every slot's weight and token number; rows behind `keep` that stay are moved.  Weights are in no order, so of n
    # slots about keep * (n - keep) / n move
    keep = case["keep"]
    moved = hk * sum(keep * (n - keep) / n for n in tokens if n > keep)
    return {"bytes": 8 * slots + 2 * moved * (4 * DIM + 8), "flops": 0}


# -- the definitions in 64 bits, request by request and head by head

def _request(s, i):
    n = int(s["lengths"][i])
    page = s["case"]["page"]
    return n, s["table"][i, :-(-n // page)].long()


def _exact_append(s):
    case = s["case"]
    hk, hq, page = case["kv_heads"], case["kv_heads"] * case["group"], case["page"]
    rows = s["qkv"].double().reshape(-1, hq + 2 * hk, 2, DIM // 2)
    table = s["cos_sin"].double().reshape(-1, 2, DIM // 2)
    keys, values, weight, token = s["keys"].double(), s["values"].double(), s["weight"].double(), s["token"].clone()
    turned = torch.empty_like(rows[:, :hq + hk])
    for i, axis in enumerate(s["axis_of"]):
        c, z = table[s["positions"][axis], 0, i], table[s["positions"][axis], 1, i]
        x, y = rows[:, :hq + hk, 0, i], rows[:, :hq + hk, 1, i]
        turned[:, :, 0, i] = x * c[:, None] - y * z[:, None]
        turned[:, :, 1, i] = y * c[:, None] + x * z[:, None]
    turned = turned.reshape(-1, hq + hk, DIM)
    first = s["row_start"].tolist()
    for b in range(case["batch"]):
        r = torch.arange(first[b], first[b + 1], device="cuda")
        slot = int(s["lengths"][b]) + r - first[b]
        at, inside = s["table"][b].long()[torch.div(slot, page, rounding_mode="floor")], slot % page
        for h in range(hk):
            keys[at, h, inside] = turned[r, hq + h]
            values[at, h, inside] = rows[r, hq + hk + h].reshape(-1, DIM)
            weight[at, h, inside] = 0.0
            token[at, h, inside] = (int(s["seen"][b]) + r - first[b]).to(torch.int32)
    return {"q": turned[:, :hq].contiguous(), "keys": keys, "values": values, "weight": weight, "token": token}


def _exact_attention(s, causal):
    """(outputs, log-sum-exp, weights) of every query row over its request's slots."""
    case, q = s["case"], s["q"].double()
    b, w, hq, _ = q.shape
    hk, group = case["kv_heads"], case["group"]
    out, lse = torch.zeros_like(q), torch.full((b, w, hq), -math.inf, dtype=torch.float64, device="cuda")
    weight = s["weight"].double()
    for i in range(b):
        n, ids = _request(s, i)
        if n == 0:
            continue
        for h in range(hk):
            k, v = (s[x][ids, h].reshape(-1, DIM)[:n].double() for x in ("keys", "values"))
            given = torch.zeros(n, dtype=torch.float64, device="cuda")
            for j in range(w):
                count = n - w + 1 + j if causal else n
                if count <= 0:
                    continue
                heads = slice(h * group, (h + 1) * group)
                z = (q[i, j, heads] @ k[:count].t()) * DIM ** -0.5
                lse[i, j, heads] = torch.logsumexp(z, 1)
                p = torch.softmax(z, 1)
                given[:count] += p.sum(0)
                if not causal:
                    out[i, j, heads] = p @ v
            full = torch.zeros(ids.numel() * case["page"], dtype=torch.float64, device="cuda")
            full[:n] = given
            weight[ids, h] += full.view(-1, case["page"])
    return out, lse[:, 0], weight


def _exact_evict(s):
    case = s["case"]
    hk, page, keep = case["kv_heads"], case["page"], case["keep"]
    keys, values = s["keys"].double(), s["values"].double()
    weight, token = s["before"][0].view(torch.float32).double(), s["before"][1].clone()
    for b in range(case["batch"]):
        n, ids = _request(s, b)
        if n <= keep:
            continue
        newest = int(s["seen"][b])
        for h in range(hk):
            w, t = weight[ids, h].reshape(-1)[:n].cpu().numpy(), token[ids, h].reshape(-1)[:n].cpu().numpy()
            safe = (t < case["sink"]) | (t >= newest - case["recent"])
            ranked = sorted(range(n), key=lambda j: (not safe[j], 0.0 if safe[j] else -w[j], j))
            stay = set(ranked[:keep])
            moves = list(zip([j for j in range(keep) if j not in stay], sorted(j for j in stay if j >= keep)))
            if not moves:
                continue
            to, of = torch.tensor(moves, device="cuda").t()
            for pool in (keys, values, weight, token):
                pool[ids[to // page], h, to % page] = pool[ids[of // page], h, of % page]
    return {"keys": keys, "values": values, "weight": weight, "token": token}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "evict":
        return _exact_evict(s)
    out, lse, weight = _exact_attention(s, case["kind"] == "observe")
    if case["kind"] == "observe":
        return weight
    found = {"out": out, "lse": lse}
    if case["weights"]:
        found["weight"] = weight
    return found
