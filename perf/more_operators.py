"""More operators around a paged KV cache, as measurable cases: what a model needs whose queries and keys are normalised, whose layers
look back over a window, and whose requests begin with the same long prompt.

All through ``retrievalattention_b200.paged``, on one cache layer: pools of pages ``[pages, kv_heads, page, 128]`` for keys and values,
a page table and a length for each request.

* ``append``  ``rope_paged_append`` with ``q_norm`` and ``k_norm``: an RMS norm of every query and key head in the pass that rotates
              them and writes keys and values to their pages;
* ``prompt``  ``paged_prompt``: attention of several new tokens of every request over the pages, causal, each token over a window of
              the last slots and a few first ones;
* ``step``    ``paged_decode`` with ``window`` and ``sink``: the same for one new token of every request;
* ``shared``  ``paged_shared_decode``: one new token of every request, where groups of requests have their first slots in common.

The plain forms are elementary torch operations in 32 bits.  Page 0 of a pool belongs to no request; page tables are filled up with it.
"""
import math

import torch

own = False

DIM = 128
THETA = 1e6
EPS = 1e-6
STALE = 0.25                             # scale of what lies in slots that no request uses
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # -- append with norms.  `tokens` rows of the longest request, `least` of the shortest; `held`: tokens already cached
        # a decode step of four requests: launches count
        dict(name="append-step-b4", kind="append", batch=4, kv_heads=8, group=4, tokens=1, least=1, held=2000, page=16,
             sections="64", interleaved=False, per_head=False, dtype="bf16"),
        # three prompts with images, of odd lengths, behind a system prompt; seven query heads a group, a weight for each head
        dict(name="append-ragged-b3", kind="append", batch=3, kv_heads=4, group=7, tokens=5001, least=77, held=333, page=32,
             sections="24,20,20", interleaved=True, per_head=True, dtype="fp16"),
        # one long prompt
        dict(name="append-32k", kind="append", batch=1, kv_heads=8, group=4, tokens=32768, least=32768, held=0, page=64,
             sections="64", interleaved=False, per_head=False, dtype="bf16"),
        # -- prompt.  `tokens` new tokens of the longest request, `least` of the shortest, behind `held` cached ones
        # pieces of prompts beside each other in a serving step
        dict(name="prompt-pieces-b4", kind="prompt", batch=4, kv_heads=8, group=4, tokens=256, least=33, held=6000, window=1024, sink=4,
             page=16, dtype="bf16"),
        # three whole prompts of odd lengths, odd window, no first tokens
        dict(name="prompt-ragged-b3", kind="prompt", batch=3, kv_heads=4, group=7, tokens=5001, least=77, held=0, window=777, sink=0,
             page=32, dtype="fp16"),
        # one long prompt
        dict(name="prompt-32k", kind="prompt", batch=1, kv_heads=8, group=4, tokens=32768, least=32768, held=0, window=2048, sink=4,
             page=64, dtype="bf16"),
        # -- step.  `tokens` slots of the longest request, `least` of the shortest
        # one user: latency
        dict(name="step-5k", kind="step", batch=1, kv_heads=8, group=4, tokens=5003, least=5003, window=1024, sink=4, page=16,
             dtype="bf16"),
        # a serving batch of uneven requests, the newest of them without a slot yet
        dict(name="step-20k-b16-ragged", kind="step", batch=16, kv_heads=4, group=7, tokens=20011, least=0, window=2000, sink=0, page=8,
             dtype="fp16"),
        # a large batch of documents, a wide window
        dict(name="step-20k-b32", kind="step", batch=32, kv_heads=8, group=4, tokens=20011, least=20011, window=8192, sink=4, page=64,
             dtype="bf16"),
        # -- shared.  `groups` of requests with `prefix` slots in common, `loose` requests with none, `tokens` to `least` slots of their own
        # a few answers to one question
        dict(name="shared-2k-b4", kind="shared", batch=4, groups=1, loose=0, kv_heads=8, group=4, prefix=2000, tokens=300, least=50,
             page=16, dtype="bf16"),
        # two system prompts, and requests without one
        dict(name="shared-6k-b24", kind="shared", batch=24, groups=2, loose=3, kv_heads=4, group=7, prefix=6016, tokens=2003, least=0,
             page=32, dtype="fp16"),
        # many questions about one long document
        dict(name="shared-32k-b64", kind="shared", batch=64, groups=1, loose=0, kv_heads=8, group=4, prefix=32768, tokens=2000, least=100,
             page=64, dtype="bf16"),
    ]


def _between(rng, low, high):
    """A whole number from low to high, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("append", "prompt", "prompt", "step", "shared", "shared"))
    kv_heads, group = rng.choice(((8, 4), (4, 7), (1, 8), (2, 8), (8, 8), (4, 1), (2, 5), (8, 2), (4, 3), (2, 6)))
    heads = kv_heads * group
    case = dict(kind=kind, kv_heads=kv_heads, group=group, page=rng.choice((8, 16, 16, 32, 64, 128, 256)),
                dtype=rng.choice(("bf16", "bf16", "fp16")))
    if kind == "append":
        step = rng.random() < 0.4
        tokens = 1 if step else _between(rng, 2, 30000 if heads <= 32 else 15000)
        case["batch"] = _between(rng, 1, 100) if step else rng.randint(1, max(1, min(6, 30000 // tokens)))
        case["held"] = rng.choice((0, _between(rng, 1, 4000)))
        case["sections"], case["interleaved"] = rng.choice((("64", False), ("16,24,24", False), ("24,20,20", True), ("32,32", False)))
        case["per_head"] = rng.random() < 0.5
        case["tokens"], case["least"] = tokens, rng.choice((tokens, rng.randint(1, tokens)))
    elif kind == "prompt":
        tokens = _between(rng, 1, 16000)
        case["batch"] = rng.randint(1, max(1, min(8, 16000 // tokens)))
        case["held"] = rng.choice((0, 0, _between(rng, 1, 16000)))
        case["sink"] = rng.choice((0, 1, 4, _between(rng, 1, 300)))
        slots = tokens + case["held"]
        case["window"] = _between(rng, 1, 4096)
        if rng.random() < 0.25 and case["batch"] * tokens * slots * heads < 1 << 30:
            case["window"] = 0                              # every slot up to the token's own
        case["tokens"], case["least"] = tokens, rng.choice((tokens, rng.randint(1, tokens)))
    elif kind == "step":
        tokens = _between(rng, 1, 60000)
        case["batch"] = _between(rng, 1, max(1, min(64, (1 << 22) // (tokens * kv_heads))))
        case["window"], case["sink"] = _between(rng, 1, 8192), rng.choice((0, 1, 4, _between(rng, 1, 300)))
        case["tokens"], case["least"] = tokens, rng.choice((tokens, rng.randint(0, tokens)))
    else:
        prefix = _between(rng, 8, 60000)
        case["batch"] = _between(rng, 2, max(2, min(64, (1 << 26) // (prefix * heads))))
        case["groups"] = rng.randint(1, max(1, min(4, case["batch"] // 2)))
        case["loose"] = rng.choice((0, 0, rng.randint(0, max(0, case["batch"] - 2 * case["groups"]))))
        case["prefix"] = -(-prefix // case["page"]) * case["page"]
        case["tokens"] = _between(rng, 1, max(2, min(4000, (1 << 20) // (case["batch"] * kv_heads))))
        case["least"] = rng.choice((case["tokens"], rng.randint(0, case["tokens"])))
    return case


def _spread(case):
    """Tokens of every request: from `tokens` (first request) to `least` (last one)."""
    b = case["batch"]
    return [case["tokens"]] if b == 1 else [case["tokens"] - (case["tokens"] - case["least"]) * i // (b - 1) for i in range(b)]


def _members(case):
    """Where the groups' requests begin: group i has requests start[i] to start[i + 1] - 1; those behind the last group have none."""
    grouped = case["batch"] - case["loose"]
    return [grouped * i // case["groups"] for i in range(case["groups"] + 1)]


def _in_common(case):
    """Slots that every request has in common with others."""
    if case["kind"] != "shared":
        return [0] * case["batch"]
    return [case["prefix"] if i < _members(case)[-1] else 0 for i in range(case["batch"])]


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
    gen.manual_seed(seed * 7919 + 3)
    kind, dtype, b, hk, page = case["kind"], DTYPES[case["dtype"]], case["batch"], case["kv_heads"], case["page"]
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    tokens, common, held, hq = _spread(case), _in_common(case), case.get("held", 0), hk * case["group"]
    used = [-(-(c + n + held) // page) for n, c in zip(tokens, common)]        # pages of every request
    numbers, pages = torch.zeros((b, max(1, max(used))), dtype=torch.long), 1
    for i, n in enumerate(used):
        first = max([m for m in _members(case) if m <= i]) if common[i] else i      # the request that has them in common with this one
        shared = common[i] // page if first != i else 0
        numbers[i, :shared] = numbers[first, :shared]
        numbers[i, shared:n] = torch.arange(pages, pages + n - shared)
        pages += n - shared
    pages += 3
    order = torch.cat((torch.zeros(1, dtype=torch.long, device="cuda"), torch.randperm(pages - 1, generator=gen, device="cuda") + 1))
    table = order[numbers.cuda()].to(torch.int32)
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
    rows = b if kind in ("step", "shared") else sum(tokens)
    state = dict(case=case, keys=keys, values=values, table=table)
    state["row_start"] = torch.tensor([0] + tokens, device="cuda").cumsum(0).to(torch.int32)
    if kind == "append":
        axis_of = _axis_of(case)
        axes = max(axis_of) + 1
        state["qkv"] = randn(rows, (hq + 2 * hk) * DIM).mul_(1 + randn(rows, 1).abs()).to(dtype)
        positions = [_image_positions(n, axes) if n > 1 else torch.full((axes, 1), 900 + i, device="cuda") for i, n in enumerate(tokens)]
        state["positions"] = torch.cat(positions, 1).long().contiguous()
        most = held + max(max(tokens), 1000) + 1000
        freq = torch.outer(torch.arange(most, dtype=torch.float32, device="cuda"),
                           1.0 / THETA ** (torch.arange(0, DIM, 2, dtype=torch.float32, device="cuda") / DIM))
        state["cos_sin"] = torch.cat((freq.cos(), freq.sin()), -1).contiguous()
        state["axis_of"] = axis_of
        state["q"] = torch.zeros((rows, hq, DIM), dtype=dtype, device="cuda")
        state["lengths"] = torch.full((b,), held, dtype=torch.int32, device="cuda")
        for name, heads in (("q_norm", hq), ("k_norm", hk)):
            state[name] = (1 + 0.3 * randn(*((heads, DIM) if case["per_head"] else (DIM,)))).to(dtype)
        return state
    state["lengths"] = torch.tensor([c + n + held for n, c in zip(tokens, common)], dtype=torch.int32, device="cuda")
    state["q"] = randn(rows, hq, DIM).to(dtype)
    if kind != "prompt":
        state["q"] = state["q"][:, None]
    if kind == "shared":
        # requests group_start[i] to group_start[i + 1] - 1 have their first shared[i] slots in common
        state["group_start"] = torch.tensor(_members(case), dtype=torch.int32, device="cuda")
        state["shared"] = torch.full((case["groups"],), case["prefix"], dtype=torch.int32, device="cuda")
    return state


def _plain_append(s):
    qkv, table, keys, values = s["qkv"], s["table"], s["keys"], s["values"]
    rows, hq, hk, page = qkv.shape[0], s["q"].shape[1], keys.shape[1], keys.shape[2]
    axis_of = torch.tensor(s["axis_of"], device="cuda")
    angle = s["cos_sin"][s["positions"]]                              # [axes, rows, 128]
    i = torch.arange(DIM // 2, device="cuda")
    cos, sin = angle[axis_of, :, i].t()[:, None], angle[axis_of, :, DIM // 2 + i].t()[:, None]
    x = qkv.view(rows, hq + 2 * hk, DIM)
    heads = x[:, :hq + hk].float()
    heads = heads * torch.rsqrt(heads.square().mean(-1, keepdim=True) + EPS)
    scale = torch.cat((s["q_norm"].float().expand(hq, DIM), s["k_norm"].float().expand(hk, DIM)))
    heads = heads * scale
    a, b = heads[..., :DIM // 2], heads[..., DIM // 2:]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(qkv.dtype)
    s["q"].copy_(turned[:, :hq])
    row = torch.arange(rows, device="cuda")
    request = torch.searchsorted(s["row_start"].long(), row, right=True) - 1
    slot = s["lengths"].long()[request] + row - s["row_start"].long()[request]
    at = table.long()[request, slot // page]
    keys[at, :, slot % page] = turned[:, hq:]
    values[at, :, slot % page] = x[:, hq + hk:]
    return {"q": s["q"], "keys": keys, "values": values}


def _rows_at(pool, table, slot):
    """The rows of slots [batch, ...] of every request, in 32 bits: [batch, heads, ..., 128]."""
    page = pool.shape[2]
    flat = slot.reshape(slot.shape[0], -1)
    id = table.long().gather(1, flat // page)
    return pool[id, :, flat % page].transpose(1, 2).reshape(slot.shape[0], pool.shape[1], *slot.shape[1:], DIM).float()


def _softmax(s):
    """Softmax over the last dimension, and its log-sum-exp; rows of -infinity are zero."""
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(m), m, 0.0))
    total = e.sum(-1, keepdim=True)
    lse = torch.where(total > 0, m + torch.log(total), float("-inf"))[..., 0]
    return e.div_(torch.where(total > 0, total, 1.0)), lse


def _plain_window(s, most):
    """Up to `most` new tokens of every request over their window and first slots; block by block of tokens, all blocks at once."""
    case, table, page = s["case"], s["table"], s["case"]["page"]
    hk, group, lengths = case["kv_heads"], case["group"], s["lengths"].long()
    q = s["q"].reshape(-1, hk, group, DIM)
    b = lengths.shape[0]
    if case["kind"] == "step":
        first_row, count = torch.arange(b, device="cuda"), torch.ones_like(lengths)
    else:
        first_row, count = s["row_start"].long()[:-1], s["row_start"].long().diff()
    window = case["window"] or table.shape[1] * page
    block = min(512, most) if case["window"] else most
    blocks = -(-most // block)
    token = torch.arange(blocks * block, device="cuda").view(blocks, block)
    inside = token < count[:, None, None]                                             # [batch, blocks, block]
    row = torch.where(inside, first_row[:, None, None] + token, 0)
    slot = (lengths - count)[:, None, None] + token                                   # a token's own
    span = window + block - 1
    seen = slot[:, :, :1] - (window - 1) + torch.arange(span, device="cuda")          # [batch, blocks, span]
    last = lengths[:, None, None] - 1
    first = torch.arange(case["sink"], device="cuda").expand(b, blocks, -1)
    seen = torch.cat((seen, first), -1)
    # of the span a token sees its window, of the first slots those in front of it
    own_slot, other = slot[..., None], seen[:, :, None]
    visible = (other >= 0) & (other <= torch.minimum(own_slot, last[..., None])) & \
        torch.where(torch.arange(seen.shape[-1], device="cuda") < span, other > own_slot - window, other <= own_slot - window)
    at = seen.clamp(min=0).minimum(last.clamp(min=0))
    k, v = _rows_at(s["keys"], table, at), _rows_at(s["values"], table, at)           # [batch, kv_heads, blocks, span, 128]
    mine = q[row].permute(0, 3, 1, 4, 2, 5).reshape(b, hk, blocks, group * block, DIM).float() / math.sqrt(DIM)
    scores = torch.matmul(mine, k.transpose(-1, -2)).view(b, hk, blocks, group, block, -1)
    scores.masked_fill_(~visible[:, None, :, None], float("-inf"))
    p, lse = _softmax(scores)
    out = torch.matmul(p.view(b, hk, blocks, group * block, -1), v).view(b, hk, blocks, group, block, DIM)
    row = torch.arange(s["q"].shape[0], device="cuda")
    request = torch.searchsorted(first_row, row, right=True) - 1
    at = request, row - first_row[request]
    out = out.permute(0, 2, 4, 1, 3, 5).reshape(b, blocks * block, hk * group, DIM)[at]
    lse = lse.permute(0, 2, 4, 1, 3).reshape(b, blocks * block, hk * group)[at]
    return {"out": out.to(q.dtype).view(s["q"].shape), "lse": lse}


def _plain_shared(s, most):
    """The scores of a group's requests over what they have in common in one product, those over up to `most` slots of their own."""
    case, table, lengths = s["case"], s["table"], s["lengths"].long()
    b, hk, group, groups, prefix = case["batch"], case["kv_heads"], case["group"], case["groups"], case["prefix"]
    starts, shared = s["group_start"].long(), s["shared"].long()
    bounds = _members(case)
    members = max(j - i for i, j in zip(bounds, bounds[1:]))                          # of the largest group
    q = s["q"].view(b, hk, group, DIM).float() / math.sqrt(DIM)
    request = torch.arange(b, device="cuda")
    mine = torch.searchsorted(starts, request, right=True) - 1
    loose = mine >= groups
    mine = mine.clamp(max=groups - 1)
    place = torch.where(loose, 0, request - starts[mine])                             # in its group
    padded = (starts[:-1, None] + torch.arange(members, device="cuda")).clamp(max=b - 1)
    slot = torch.arange(prefix, device="cuda").expand(groups, prefix)
    k, v = (_rows_at(s[x], table[starts[:-1]], slot) for x in ("keys", "values"))     # [groups, kv_heads, prefix, 128]
    first = torch.matmul(q[padded].transpose(1, 2).reshape(groups, hk, members * group, DIM), k.transpose(-1, -2))
    first = first.view(groups, hk, members, group, prefix)[mine, :, place]
    first = torch.where((loose[:, None] | (slot[0] >= shared[mine][:, None]))[:, None, None], float("-inf"), first)
    own_slot = torch.where(loose, 0, shared[mine])[:, None] + torch.arange(most, device="cuda")
    at = own_slot.minimum((lengths - 1).clamp(min=0)[:, None])
    own_k, own_v = (_rows_at(s[x], table, at) for x in ("keys", "values"))
    second = torch.matmul(q, own_k.transpose(-1, -2))
    second = torch.where((own_slot < lengths[:, None])[:, None, None], second, float("-inf"))
    p, lse = _softmax(torch.cat((first, second), -1))
    given = p[padded][..., :prefix].transpose(1, 2).reshape(groups, hk, members * group, prefix)
    out = torch.matmul(given, v).view(groups, hk, members, group, DIM)[mine, :, place]
    out = torch.where(loose[:, None, None, None], 0.0, out) + torch.matmul(p[..., prefix:], own_v)
    return {"out": out.reshape(b, 1, hk * group, DIM).to(s["q"].dtype), "lse": lse.reshape(b, hk * group)}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "append":
            return _plain_append(s)
        most = max(1, case["tokens"])
        return _plain_shared(s, most) if kind == "shared" else _plain_window(s, most if kind == "prompt" else 1)
    from retrievalattention_b200 import paged
    if kind == "append":
        paged.rope_paged_append(s["qkv"], s["cos_sin"], s["positions"], s["axis_of"], s["q"], s["keys"], s["values"], s["table"],
                                s["lengths"], s["row_start"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return {"q": s["q"], "keys": s["keys"], "values": s["values"]}
    lse = torch.empty((s["q"].shape[0], s["q"].shape[-2]), dtype=torch.float32, device="cuda")
    cache = s["q"], s["keys"], s["values"], s["table"], s["lengths"]
    if kind == "prompt":
        out = paged.paged_prompt(*cache, s["row_start"], window=case["window"] or None, sink=case["sink"], lse=lse)
    elif kind == "step":
        out = paged.paged_decode(*cache, window=case["window"], sink=case["sink"], lse=lse)
    else:
        out = paged.paged_shared_decode(*cache, s["group_start"], s["shared"], lse=lse)
    return {"out": out, "lse": lse}


def _visible(case, n, count):
    """Pairs of a token and a slot that it sees, and slots that some token sees, for the last `count` tokens of n."""
    window, sink = case["window"] or n, case["sink"]
    pairs = 0
    for own_slot in range(n - count, n):
        low = max(0, own_slot - window + 1)
        pairs += own_slot + 1 - low + min(sink, low)
    low = max(0, n - count - window + 1)
    return pairs, n - low + min(sink, low)


def work(case):
    kind, hk, tokens = case["kind"], case["kv_heads"], _spread(case)
    hq = hk * case["group"]
    if kind == "append":
        rows, heads = sum(tokens), hq + 2 * hk
        axes = len(case["sections"].split(","))
        # the projection in, queries and cache rows out, a table row and the positions in
        return {"bytes": rows * (2 * heads * DIM * 2 + 4 * DIM + 8 * axes), "flops": rows * (heads - hk) * DIM * 7}
    if kind == "shared":
        members = _members(case)[-1]
        slots, pairs = sum(tokens) + case["groups"] * case["prefix"], sum(tokens) + members * case["prefix"]
        return {"bytes": slots * hk * 4 * DIM + case["batch"] * hq * (4 * DIM + 4), "flops": 4 * DIM * pairs * hq}
    counts = tokens if kind == "prompt" else [min(1, n) for n in tokens]
    seen = [_visible(case, n + case.get("held", 0), c) for n, c in zip(tokens, counts)]
    rows = sum(tokens) if kind == "prompt" else case["batch"]
    return {"bytes": sum(s for _, s in seen) * hk * 4 * DIM + rows * hq * (4 * DIM + 4), "flops": 4 * DIM * sum(p for p, _ in seen) * hq}


# -- the definitions in 64 bits, request by request and head by head

def _exact_append(s):
    case = s["case"]
    hk, hq, page = case["kv_heads"], case["kv_heads"] * case["group"], case["page"]
    rows = s["qkv"].double().reshape(-1, hq + 2 * hk, DIM)
    normed = torch.empty_like(rows[:, :hq + hk])
    for h in range(hq + hk):
        x = rows[:, h]
        scale = s["q_norm"] if h < hq else s["k_norm"]
        if scale.dim() == 2:
            scale = scale[h if h < hq else h - hq]
        normed[:, h] = x / torch.sqrt((x * x).sum(-1, keepdim=True) / DIM + EPS) * scale.double()
    halves, turned = normed.reshape(-1, hq + hk, 2, DIM // 2), torch.empty_like(normed).reshape(-1, hq + hk, 2, DIM // 2)
    table = s["cos_sin"].double().reshape(-1, 2, DIM // 2)
    for i, axis in enumerate(s["axis_of"]):
        c, z = table[s["positions"][axis], 0, i], table[s["positions"][axis], 1, i]
        x, y = halves[:, :, 0, i], halves[:, :, 1, i]
        turned[:, :, 0, i] = x * c[:, None] - y * z[:, None]
        turned[:, :, 1, i] = y * c[:, None] + x * z[:, None]
    turned = turned.reshape(-1, hq + hk, DIM)
    keys, values = s["keys"].double(), s["values"].double()
    first = s["row_start"].tolist()
    for b in range(case["batch"]):
        r = torch.arange(first[b], first[b + 1], device="cuda")
        slot = int(s["lengths"][b]) + r - first[b]
        at, inside = s["table"][b].long()[torch.div(slot, page, rounding_mode="floor")], slot % page
        for h in range(hk):
            keys[at, h, inside] = turned[r, hq + h]
            values[at, h, inside] = rows[r, hq + hk + h]
    return {"q": turned[:, :hq].contiguous(), "keys": keys, "values": values}


def _exact_attention(s):
    """Every query row over the slots that it sees, in runs of tokens."""
    case, kind = s["case"], s["case"]["kind"]
    q = s["q"].double().reshape(-1, case["kv_heads"] * case["group"], DIM)
    hk, group, page = case["kv_heads"], case["group"], case["page"]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    starts, lengths, table = s["row_start"].tolist(), s["lengths"].tolist(), s["table"].long()
    for b, n in enumerate(lengths):
        count, row = (starts[b + 1] - starts[b], starts[b]) if kind == "prompt" else (1, b)
        window, sink = (n, 0) if kind == "shared" else (case["window"] or n, case["sink"])
        for t in range(0, count if n else 0, 512):
            own_slot = torch.arange(n - count + t, n - count + min(t + 512, count), device="cuda")
            low = max(0, int(own_slot[0]) - window + 1)
            slots = torch.cat((torch.arange(min(sink, low), device="cuda"), torch.arange(low, int(own_slot[-1]) + 1, device="cuda")))
            sees = (slots <= own_slot[:, None]) & ((slots > own_slot[:, None] - window) | (slots < sink))
            at, inside = table[b, torch.div(slots, page, rounding_mode="floor")], slots % page
            r = slice(row + t, row + t + own_slot.numel())
            for h in range(hk):
                k, v = s["keys"][at, h, inside].double(), s["values"][at, h, inside].double()
                z = torch.einsum("tgd,sd->tgs", q[r, h * group:(h + 1) * group], k) * DIM ** -0.5
                z = z.masked_fill(~sees[:, None], -math.inf)
                lse[r, h * group:(h + 1) * group] = torch.logsumexp(z, -1)
                out[r, h * group:(h + 1) * group] = torch.einsum("tgs,sd->tgd", torch.softmax(z, -1), v)
    return {"out": out.reshape(s["q"].shape), "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attention(s)
