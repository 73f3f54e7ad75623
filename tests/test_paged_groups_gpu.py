"""``paged_cache.attend`` of some of the requests, some of which begin alike, against attention of each by itself in 64 bits."""
import pytest
import torch

from attend_helpers import attend_rows, close
from paged_helpers import DIM

pytestmark = pytest.mark.gpu


def filled(cache, gen):
    """Random keys and values in the whole pool."""
    for pool in (cache.key_pages[0], cache.value_pages[0]):
        pool.copy_(torch.randn(pool.shape, generator=gen, device="cuda"))


def slots(cache, pool, b):
    n = cache.length_of[b]
    x = pool[torch.tensor(cache._pages[b], device="cuda")].transpose(0, 1).reshape(pool.shape[1], -1, DIM)
    return x[:, :n].double().cpu()


def check(cache, q, out, lse, requests):
    for i, b in enumerate(requests):
        k, v = (slots(cache, x[0], b) for x in (cache.key_pages, cache.value_pages))
        want = attend_rows(q[i].double().cpu(), k, v, torch.ones(1, k.shape[1], dtype=torch.bool))
        assert close(out[i], lse[i:i + 1], *want), b


def test_requests_that_run_on(monkeypatch):
    """Nested prompts, one request done, another one of its own in a place between; the shared kernels run (the table has room for many slots)."""
    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors
    from retrievalattention_b200.cache_hub import paged_cache

    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    hk, batch, common = 2, 24, 24000
    cache = paged_cache(1, batch, 30000, hk, 8, DIM, torch.bfloat16, {"0": "cuda:0"}, 1, 1, page_size=64, num_pages=600)
    filled(cache, gen)
    cache.begin([70] + [0] * (batch - 1))
    assert cache.share(0, [1]) == 64
    cache.begin([0, common] + [0] * (batch - 2))
    n = cache.share(1, list(range(2, batch)))
    assert n == common + 64 - common % 64
    cache.begin([3, 5] + [i % 7 for i in range(2, batch)])
    shared_calls, shared_decode = [], paged.paged_shared_decode
    monkeypatch.setattr(paged, "paged_shared_decode", lambda *args, **rest: shared_calls.append(args[5:7]) or shared_decode(*args, **rest))
    for done in (None, 5, 1, 0, 23):
        if done is not None:
            cache.release(done)
        running = [b for b in range(batch) if cache.length_of[b]]
        cache.begin([1 if cache.length_of[b] else 0 for b in range(batch)])
        q = torch.randn((len(running), 1, 8, DIM), generator=gen, device="cuda").to(torch.bfloat16)
        lse = torch.empty(len(running), 8, device="cuda")
        out = cache.attend(q, 0, lse=lse, requests=None if len(running) == batch else running)
        check_prefill_errors()
        check(cache, q, out, lse, running)
    assert len(shared_calls) == 5
    assert [x[1].max().item() for x in shared_calls] == [n] * 5


def test_a_model_whose_requests_begin_alike(monkeypatch):
    """Prompts, a nested prefix, steps, and requests that are done, over the kernels that read once what is in common (whole page tables, and
    whatever that saves), against the model in 32 bits."""
    from test_paged_layers_gpu import check as check_model, small

    from retrievalattention_b200 import paged
    from retrievalattention_b200.attn_hub.retroinfer_attn import check_prefill_errors

    model = small((None, 24), batch=5, max_length=120000)
    cache = model.cache
    rows = lambda requests: slice(None) if requests is None else torch.tensor(requests, device="cuda")  # noqa: E731
    monkeypatch.setattr(cache, "_of", lambda requests: (cache.page_table[rows(requests)], cache.lengths[rows(requests)]))
    for name in ("_PAYS_MB", "_PAYS_MB_EACH"):
        monkeypatch.setattr(cache, name, 0)
    calls, shared_decode = [], paged.paged_shared_decode
    monkeypatch.setattr(paged, "paged_shared_decode", lambda *args, **rest: calls.append(args[6].tolist()) or shared_decode(*args, **rest))
    gen = torch.Generator().manual_seed(2)
    prompt = lambda n: torch.randint(0, 1000, (n,), generator=gen).cuda()  # noqa: E731
    begin, document = prompt(35), prompt(150)
    for b in range(1, 5):
        model.release(b)
    ids = [list(begin), None, None, None, None]
    check_model(model, model.prefill_forward([begin], requests=[0]), ids, (0,))
    assert model.share(0, [1]) == 32
    ids[1] = list(begin[:32]) + list(document)
    check_model(model, model.extend_forward([document], requests=[1]), ids, (1,))
    assert model.share(1, [2, 3], 182) == 176
    rest = [torch.cat([document[144:], prompt(n)]) for n in (3, 20)]
    for b, p in zip((2, 3), rest):
        ids[b] = list(begin[:32]) + list(document[:144]) + list(p)
    check_model(model, model.extend_forward(rest, requests=[2, 3]), ids, (2, 3))
    other = prompt(40)
    ids[4] = list(other)
    check_model(model, model.prefill_forward([other], requests=[4]), ids, (4,))
    for done in (None, 2, 0):
        if done is not None:
            model.release(done)
        running = [b for b in range(5) if b not in model._released]
        for _ in range(3):
            check_model(model, model.decode_forward(), ids, running)
    check_prefill_errors()
    # of layers without a window: groups of all, of 0, 1, 3, 4 and of 1, 3, 4
    assert calls == [[0, 176, 0, 0, 0]] * 3 + [[0, 176, 0]] * 3 + [[176, 0]] * 3
