"""The host side of steps of packed requests where it can go wrong, without a GPU: launches of empty steps, sizes of
workspaces, and the decoder's bookkeeping."""
from types import SimpleNamespace

import pytest
import torch

from mlx_gsq_amd.models import PackedGraphDecoder, build_qwen35
from qwen35_fixture import ARGS, TinyStore, dense_factories
from test_host_launches import run, stub  # noqa: F401  (a fixture)
from test_paged_launches import SIGNATURES


# ---- launches and workspaces ---------------------------------------------------------------------


def test_no_launch_is_empty(stub):  # noqa: F811
    """A step without sequences has no workgroup to give a launch over sequences: the convolution and the launch that
    clears the rows run, as many as with a hint of single tokens."""
    run(stub, SIGNATURES + """
for tokens in (1, 16, 100, 5000):
    for most in (None, 1):
        before = stub.stub_launches()
        assert gdn(tokens, 0, most) == 0 and stub.stub_launches() - before == 2, (tokens, most)
    assert lib.gsq_gdn_packed_work(tokens, 0, 16, 48, 128, 128, 4, tokens) == lib.gsq_gdn_packed_work(tokens, 0, 16, 48, 128, 128, 4, 1)
    assert attn(tokens, 0, 80) == 0
""")


def test_workspaces_do_not_grow_with_single_tokens(stub):  # noqa: F811
    """T, P and gates of a chunk are kept for sequences that go by chunks, of which a step of N tokens has N / 16 at most:
    what 251 sequences with one turn of 16 among them take is what 16 take, and their own rows."""
    run(stub, SIGNATURES + """
def floats(tokens, sequences, most=None):
    return lib.gsq_gdn_packed_work(tokens, sequences, 16, 48, 128, 128, 4, tokens if most is None else most)
rows = 10240 + 48 * 128  # of a token: convolution and recurrence outputs
chunk = 48 * (2 * 64 * 64 + 3 * 64)  # of a chunk
for tokens, sequences in ((266, 251), (1050, 1024), (1024, 1024), (16, 1), (64, 4), (2047 * 3, 3), (524280, 1024)):
    got = floats(tokens, sequences)
    assert got == tokens * rows + (tokens // 64 + min(sequences, tokens // 16) + 1) * chunk, (tokens, sequences, got)
assert floats(266, 251) * 4 < 60 << 20
assert floats(1050, 1024) * 4 < 230 << 20
# what the chunks of any step take: sequences of 16 and more and shorter ones in all orders
import random
rng = random.Random(5)
for _ in range(2000):
    new = [rng.choice([0, 1, 15, 16, 17, 63, 64, 65, 80, 200]) for _ in range(rng.randint(1, 40))]
    tokens, at, longs, last = sum(new), 0, 0, -1
    if not tokens:
        continue
    for n in new:
        if n >= 16:
            first, chunks = at // 64 + longs, -(-n // 64)
            assert first > last  # no two chunks share a slot
            last = first + chunks - 1
            longs += 1
        at += n
    assert last < tokens // 64 + min(len(new), tokens // 16) + 1
""")


# ---- the decoder ---------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def model():
    store = TinyStore("cpu", seed=1)
    linear, fused, embedding = dense_factories(store)
    return build_qwen35(store, dtype=torch.float32, args=ARGS, linear=linear, fused=fused, embedding=embedding)


def test_a_step_that_fails_part_way_cannot_be_repeated(model, monkeypatch):
    """Layers before the failure have advanced their requests' states: every step is refused until those are released."""
    with torch.no_grad():
        cache = model.new_paged_cache(4, pages=8, page_size=16, max_len=32)
        model.step([5, 6, 7, 8], [3, 1], [2, 0], cache)
        want = model.new_paged_cache(4, pages=8, page_size=16, max_len=32)
        want = model.step([9, 10, 11], [2, 1], [3, 2], want)
        before = {i: t.clone() for i, t in cache.rec.items()}

        def fail(*_):
            raise MemoryError("no room")
        for last in (model.layers[-1], model.lm_head):
            with monkeypatch.context() as m:
                m.setattr(last, "forward", fail)
                with pytest.raises(MemoryError):
                    model.step([9, 10], [1, 1], [2, 0], cache)
            assert any(not torch.equal(t, before[i]) for i, t in cache.rec.items()) and cache.lengths.tolist() == [1, 0, 3, 0]
            decoder = object.__new__(PackedGraphDecoder)
            decoder.cache, decoder.batch = cache, 4
            for _ in range(2):
                for call in (lambda: model.step([9, 10], [1, 1], [2, 0], cache), lambda: model.step([9], [1], [3], cache),
                             lambda: decoder.step([9], [2])):
                    with pytest.raises(ValueError, match="failed part way"):
                        call()
                cache.release([0])
            cache.release([1, 2])
            assert int(cache.n_free) == 8
            got = model.step([9, 10, 11], [2, 1], [3, 2], cache)  # new requests begin from zeros
            assert torch.equal(got, want)
            cache.release(torch.arange(4))
            model.step([5, 6, 7, 8], [3, 1], [2, 0], cache)


def test_a_step_that_is_refused_leaves_a_cache_whole(model):
    with torch.no_grad():
        cache = model.new_paged_cache(2, pages=2, page_size=16, max_len=32)
        for args in (([1, 2], [1], [0]), ([], [], []), ([1], [1], [5])):
            with pytest.raises(ValueError):
                model.step(*args, cache)
        assert cache.torn is None and bool(torch.isfinite(model.step([1, 2], [2], [0], cache)).all())


def test_a_step_that_served_nobody_leaves_a_cache_whole(model, monkeypatch):
    with torch.no_grad():
        cache = model.new_paged_cache(2, pages=2, page_size=16, max_len=32)
        with monkeypatch.context() as m:
            m.setattr(model.lm_head, "forward", lambda *_: 1 / 0)
            with pytest.raises(ZeroDivisionError):
                model.step([1] * 33, [33], [0], cache)  # longer than max_len
        assert bool(torch.isfinite(model.step([1, 2], [2], [0], cache)).all())


def test_request_numbers_past_32_bits_are_out_of_range(model):
    """2^32 + 1 is not request 1."""
    far = [2 ** 32 + 1, 2 ** 31 + 1, -2 ** 32 + 1, -2 ** 40]
    with torch.no_grad():
        cache = model.new_paged_cache(2, pages=2, page_size=16, max_len=32)
        model.step([1, 2], [2], [1], cache)
        for some in (torch.tensor(far), far, torch.tensor(far[:1])):
            cache.release(some)
            assert cache.lengths.tolist() == [0, 2] and int(cache.n_free) == 1
        with pytest.raises(ValueError, match="whole numbers"):
            cache.release([1.0])
        decoder = object.__new__(PackedGraphDecoder)
        decoder.cache, decoder.batch, decoder.logits, decoder.graph = cache, 4, torch.zeros(4, 8), SimpleNamespace(replay=lambda: None)
        decoder.ids, decoder.requests, decoder.new = torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
        decoder.step([5] * 4, torch.tensor(far))
        assert all(r < 0 or r >= cache.requests for r in decoder.requests.tolist())
        cache.release(torch.tensor([1], dtype=torch.int16))
        assert cache.lengths.tolist() == [0, 0] and int(cache.n_free) == 2
        cache.release([])


def test_max_len_is_what_a_request_may_have(model):
    """Whole pages: 17 positions in pages of 16 are 32, and a 33rd is not served."""
    with torch.no_grad():
        cache = model.new_paged_cache(1, pages=4, page_size=16, max_len=17)
        assert cache.max_len == 32 and cache.table.shape == (1, 2)
        assert bool(torch.isfinite(model.step([3] * 32, [32], [0], cache)).all())
        assert bool(torch.isnan(model.step([3], [1], [0], cache)).all()) and cache.lengths.tolist() == [32]
