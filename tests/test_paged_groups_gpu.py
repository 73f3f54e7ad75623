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
