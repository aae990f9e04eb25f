"""The Qwen3.5-hybrid decoder serving many requests at once (``new_paged_cache``, ``step``, ``PackedGraphDecoder``) against
each request run by itself.

CPU: the torch formulation in float32 on dense stand-ins. GPU: the kernels between packed projections, fp16."""
import pytest
import torch

import paged_ref as R
from mlx_gsq_amd import tables
from mlx_gsq_amd.models import PackedGraphDecoder, build_qwen35
from qwen35_fixture import ARGS, TABLES, TinyStore, dense_factories, rel_l2

A, B, C = [17, 301, 5, 77, 402, 9, 256, 130, 44, 8, 19, 350, 2, 61, 90, 111, 7, 300, 21, 45], [9, 44, 256], [81, 300, 12, 500, 3, 77, 5]


@pytest.fixture(scope="module")
def store():
    return TinyStore("cpu", seed=1)


def _cpu_model(store):
    linear, fused, embedding = dense_factories(store)
    return build_qwen35(store, dtype=torch.float32, args=ARGS, linear=linear, fused=fused, embedding=embedding)


def _gpu_model():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    tables.set_tables(TABLES)
    return build_qwen35(TinyStore(torch.device("cuda:0"), seed=1), dtype=torch.float16, args=ARGS)


def _alone(model, tokens):
    """Logits behind every token of one sequence, token by token."""
    cache = model.new_cache(max_len=64)
    return torch.cat([model(torch.tensor([[t]], device=model.norm_w.device), cache) for t in tokens], dim=1)[0]


def _close(x, y, tol):
    return rel_l2(x.float().cpu().numpy(), y.float().cpu().numpy()) <= tol


def _check_steps(model, tol):
    """Prompts, pieces and single tokens of three requests in turn, one of them over the pages that another left."""
    with torch.no_grad():
        a, b, c = (_alone(model, t) for t in (A, B, C))
        cache = model.new_paged_cache(4, pages=5, page_size=16, max_len=48)
        got = model.step(A[:9] + B[:2], [9, 2], [2, 0], cache)
        assert _close(got, torch.stack([a[8], b[1]]), tol)
        got = model.step(B[2:] + A[9:19], [1, 10], [0, 2], cache, all_logits=True)
        assert _close(got, torch.cat([b[2:], a[9:19]]), tol)
        assert cache.lengths.tolist() == [3, 0, 19, 0] and cache.held.tolist() == [1, 0, 2, 0] and int(cache.n_free) == 2
        cache.release([0, 0, 9])
        assert cache.lengths.tolist() == [0, 0, 19, 0] and int(cache.n_free) == 3
        got = model.step(C[:6] + A[19:], [6, 1], [3, 2], cache)
        assert _close(got, torch.stack([c[5], a[19]]), tol)
        got = model.step(C[6:] + B, [1, 3], [3, 0], cache)  # a request's number again, from the beginning
        assert _close(got, torch.stack([c[6], b[2]]), tol)


def _check_no_pages(model, tol):
    """A sequence that the pages do not suffice for is not served, keeps what it has, and goes on when there are some."""
    with torch.no_grad():
        a = _alone(model, A)
        cache = model.new_paged_cache(2, pages=2, page_size=16, max_len=32)
        model.step(A[:16] + B, [16, 3], [0, 1], cache)
        got = model.step([A[16], 44], [1, 1], [0, 1], cache)
        assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1]).all())
        assert cache.lengths.tolist() == [16, 4] and int(cache.n_free) == 0
        cache.release([1])
        got = model.step(A[16:], [4], [0], cache)
        assert _close(got, a[19:], tol)
        got = model.step(C + C[:6], [13], [0], cache)  # past max_len
        assert bool(torch.isnan(got).all()) and cache.lengths.tolist() == [20, 0]


def test_cpu_steps(store):
    _check_steps(_cpu_model(store), 1e-5)


def test_cpu_no_pages(store):
    _check_no_pages(_cpu_model(store), 1e-5)


def test_cpu_plan_matches_definition(store):
    model = _cpu_model(store)
    g = R.gen("host plan")
    for _ in range(30):
        cache = model.new_paged_cache(5, pages=9, page_size=16, max_len=64)
        lists = [0] * 5, [0] * 5, [[-1] * 4 for _ in range(5)], list(range(9)), 9
        lengths, held, table, free, n_free = lists
        for _ in range(6):
            n = int(torch.randint(1, 5, (1,), generator=g))
            requests = torch.randint(-1, 6, (n,), generator=g).tolist()
            new = torch.randint(-1, 30, (n,), generator=g).tolist()
            plan = cache.plan(torch.tensor(requests), torch.tensor(new), 60)
            want, n_free = R.plan(requests, new, lengths, held, table, free, n_free, 60, 16)
            assert [t.tolist() for t in plan] == list(want)
            cache.advance(plan)
            for r, x in zip(want[1], want[2]):
                if r >= 0:
                    lengths[r] = x
            back = torch.randint(-1, 6, (2,), generator=g).tolist()
            cache.release(back)
            n_free = R.release(back, lengths, held, table, free, n_free)
            assert cache.table.tolist() == table and cache.held.tolist() == held and cache.lengths.tolist() == lengths
            assert int(cache.n_free) == n_free and cache.free.tolist()[:n_free] == free[:n_free]


def test_cpu_refusals(store):
    model = _cpu_model(store)
    cache = model.new_paged_cache(3, pages=4, page_size=16, max_len=32)
    for ids, new, requests, match in (([1, 2], [1], [0], "as many tokens"), ([1, 2], [2, 0], [0, 1], "at least one"),
                                      ([1, 2], [1, 1], [1, 1], "different"), ([1], [1], [3], "below 3"), ([1], [1], [-1], "below 3"),
                                      ([1, 2], [1, 1], [0], "as many tokens"), ([], [], [], "a token at least")):
        with pytest.raises(ValueError, match=match):
            model.step(ids, new, requests, cache)
    assert cache.lengths.tolist() == [0, 0, 0] and int(cache.n_free) == 4
    for kw in (dict(page_size=8), dict(pages=0), dict(requests=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            model.new_paged_cache(**dict(dict(requests=2, pages=2, page_size=16, max_len=16), **kw))
    model.dtype = torch.float32
    with pytest.raises(ValueError, match="16-bit"):
        model.new_paged_cache(2, 2, device="cuda:0")


@pytest.mark.gpu
def test_gpu_steps():
    model = _gpu_model()
    _check_steps(model, 2e-2)
    _check_no_pages(model, 2e-2)


@pytest.mark.gpu
def test_gpu_graph_of_single_tokens():
    """Replayed steps of requests that join, grow and end are the eager steps, bit for bit."""
    model = _gpu_model()
    with torch.no_grad():
        caches = [model.new_paged_cache(5, pages=6, page_size=16, max_len=64) for _ in range(2)]
        for c in caches:
            model.step(A[:15] + C, [15, 7], [4, 1], c)
        graph = PackedGraphDecoder(model, caches[0], 4)
        assert caches[0].lengths.tolist() == caches[1].lengths.tolist() == [0, 7, 0, 0, 15]
        for ids, requests in (([3, 40], [4, 1]), ([5], [1]), ([7, 8, 9], [1, 4, 0]), ([1, 2, 3, 4], [0, 2, 4, 1]), ([6], [4])):
            got = graph.step(ids, requests).clone()
            n = len(ids)
            rows = torch.full((4,), -1, dtype=torch.int32, device=got.device)
            new = torch.zeros_like(rows)
            rows[:n], new[:n] = torch.tensor(requests, dtype=torch.int32), 1
            padded = torch.cat([torch.tensor(ids), graph.ids[n:].cpu()]).to(got.device)
            want = model.step(padded, new, rows, caches[1], max_new=1)[:n]
            assert torch.equal(got, want) and bool(torch.isfinite(got).all())
            assert caches[0].lengths.tolist() == caches[1].lengths.tolist()
            assert all(torch.equal(x, y) for x, y in zip(caches[0].rec.values(), caches[1].rec.values()))
            for c in caches:
                if requests == [1, 4, 0]:
                    c.release([4])
        with pytest.raises(ValueError, match="at most 4"):
            graph.step([1] * 5, [0, 1, 2, 3, 4])
