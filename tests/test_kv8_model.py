"""The Qwen3.5-hybrid decoder on an 8-bit K/V cache, and trees of drafted tokens through it (``verify``,
``accept``): against HF's logits, and against the same tokens decoded one at a time.

CPU: the torch formulation in float32 on dense stand-ins. GPU: the kernels (kv8_write, attn_kv8, gdn_tree,
gdn_seq) between packed projections, fp16."""
import pytest
import torch

from mlx_gsq_amd import tables
from mlx_gsq_amd.models import GraphDecoder, build_qwen35
from mlx_gsq_amd.models.qwen35 import Qwen35Cache
from qwen35_fixture import ARGS, TABLES, TinyStore, dense_factories, hf_logits, hf_model, rel_l2

IDS = [17, 301, 5, 77, 402, 9, 256, 130]
# a tree behind the first 5 tokens: two continuations, one of which branches again
DRAFT = [9, 44, 256, 130, 81, 300, 12]
PARENTS = [-1, -1, 0, 2, 2, 1, 3]
PATHS = [[0], [1], [0, 2], [0, 2, 3], [0, 2, 4], [1, 5], [0, 2, 3, 6]]


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


def _ids(model, tokens):
    return torch.tensor([tokens], device=model.norm_w.device)


def _one_at_a_time(model, tokens, batch=1):
    cache = model.new_cache(batch=batch, max_len=32, kv_bits=8)
    return torch.cat([model(_ids(model, [t]).expand(batch, 1), cache) for t in tokens], dim=1)


def _check_tree(model, tol):
    """Every node's logits are those of its path decoded one token at a time; each accepted path goes on as
    that sequence does."""
    with torch.no_grad():
        cache = model.new_cache(max_len=32, kv_bits=8)
        model(_ids(model, IDS[:5]), cache)
        before = [t.clone() for t in (*cache.rec.values(), *cache.conv.values())]
        logits = model.verify(_ids(model, DRAFT), cache, PARENTS)
        assert cache.length == 5 and int(cache.pos) == 5
        assert all(torch.equal(a, b) for a, b in zip(before, (*cache.rec.values(), *cache.conv.values())))
        for t, path in enumerate(PATHS):
            want = _one_at_a_time(model, IDS[:5] + [DRAFT[i] for i in path])[:, -1]
            assert rel_l2(logits[:, t].float().cpu().numpy(), want.float().cpu().numpy()) <= tol, t
        for path in ([0, 2, 3, 6], [1], [0, 2, 4], []):
            cache = model.new_cache(max_len=32, kv_bits=8)
            model(_ids(model, IDS[:5]), cache)
            model.verify(_ids(model, DRAFT), cache, torch.tensor(PARENTS))
            model.accept(cache, path)
            assert cache.length == int(cache.pos) == 5 + len(path)
            got = model(_ids(model, [77]), cache)[:, -1]
            want = _one_at_a_time(model, IDS[:5] + [DRAFT[i] for i in path] + [77])[:, -1]
            assert rel_l2(got.float().cpu().numpy(), want.float().cpu().numpy()) <= tol, path


def test_cpu_8_bit_cache_matches_hf(store):
    """K and V rows are off by half a step of their largest value over 127 at most: a root mean square error of
    0.3 / 127 of about three standard deviations, 0.7 per cent of a row, in one layer of four."""
    ref = hf_logits(hf_model(store), IDS)
    model = _cpu_model(store)
    with torch.no_grad():
        pre = model(_ids(model, IDS), model.new_cache(max_len=16, kv_bits=8))
        dec = _one_at_a_time(model, IDS)
    assert 1e-6 < rel_l2(pre.numpy(), ref.numpy()) <= 7e-3
    assert rel_l2(dec.numpy(), pre.numpy()) <= 1e-4


def test_cpu_tree(store):
    _check_tree(_cpu_model(store), 1e-4)


def test_cpu_trees_of_a_batch(store):
    """Rows with trees of their own, that keep different paths of one length."""
    model = _cpu_model(store)
    parents = torch.tensor([[-1, 0, 0, 2], [-1, -1, 1, 0]])
    draft = torch.tensor([[9, 44, 256, 130], [81, 300, 12, 5]])
    paths = [[0, 2, 3], [1, 2, 2]]
    with torch.no_grad():
        cache = model.new_cache(batch=2, max_len=16, kv_bits=8)
        model(torch.tensor([IDS[:4], IDS[4:]]), cache)
        logits = model.verify(draft, cache, parents)
        with pytest.raises(ValueError, match="path"):
            model.accept(cache, paths)  # token 2 does not follow itself
        paths = [[0, 2], [1, 2]]
        model.accept(cache, paths)
        nxt = model(torch.tensor([[3], [3]]), cache)[:, -1]
        for b, ids in enumerate((IDS[:4], IDS[4:])):
            seq = _one_at_a_time(model, ids + [int(draft[b, i]) for i in paths[b]] + [3])
            assert rel_l2(nxt[b].numpy(), seq[0, -1].numpy()) <= 1e-4
            assert rel_l2(logits[b, paths[b][-1]].numpy(), seq[0, -2].numpy()) <= 1e-4


def test_cpu_refusals(store):
    model = _cpu_model(store)
    with torch.no_grad():
        with pytest.raises(ValueError, match="kv_bits"):
            model.new_cache(kv_bits=4)
        with pytest.raises(ValueError, match="8-bit"):
            model.verify(_ids(model, DRAFT), model.new_cache(max_len=16), PARENTS)
        cache = model.new_cache(max_len=8, kv_bits=8)
        with pytest.raises(ValueError, match="verify"):
            model.accept(cache, [0])
        for bad in ([-1, 1, 0], [-1, 0, -2], [0, 0, 0], [-1, 0]):
            with pytest.raises(ValueError):
                model.verify(_ids(model, [1, 2, 3]), cache, bad)
        with pytest.raises(ValueError, match="64"):
            model.verify(_ids(model, [1] * 65), cache, [-1] * 65)
        with pytest.raises(ValueError, match="positions"):
            model.verify(_ids(model, [1] * 9), cache, [-1] * 9)
        model.verify(_ids(model, [1, 2, 3]), cache, [-1, 0, 0])
        for bad in ([1], [0, 1, 2], [3], [-1], [[0], [0]], [0, 0]):
            with pytest.raises(ValueError):
                model.accept(cache, bad)
        model(_ids(model, [4]), cache)  # a plain step forgets the drafted tokens
        with pytest.raises(ValueError, match="verify"):
            model.accept(cache, [0])
        cache.reset()
        assert cache.length == 0 and cache.drafted is None
        # a call that fails leaves no tree behind, the one before it included
        model.verify(_ids(model, [1, 2, 3]), cache, [-1, 0, 0])
        for ids, parents, match in ((_ids(model, [1] * 9), [-1] * 9, "positions"), (torch.tensor([[1], [2]]), [-1], "rows")):
            with pytest.raises(ValueError, match=match):
                model.verify(ids, cache, parents)
        with pytest.raises(ValueError, match="verify"):
            model.accept(cache, [0])
        # parents that the device was asked to check, and that are no tree: the cache does not hold the tokens
        model.verify(_ids(model, [1, 2, 3]), cache, [-1, 0, 0])
        cache.drafted = (torch.tensor([-1, 0, 2], dtype=torch.int32), cache.drafted[1])
        with pytest.raises(ValueError, match="no tree"):
            model.accept(cache, [0, 1])
        assert cache.length == 0
    # no derivative goes through the cache
    layer = model.layers[3].mixer
    x = torch.randn(1, 2, ARGS.hidden_size, requires_grad=True)
    with pytest.raises(ValueError, match="derivative"):
        layer(x, Qwen35Cache(ARGS, 1, 8, "cpu", torch.float32, kv_bits=8))


class _Fails(torch.nn.Module):
    def forward(self, *args, **kw):
        raise RuntimeError("out of memory")

    replay = forward


@pytest.mark.parametrize("where", ["last layer", "head", "replay"])
def test_cpu_failed_step_leaves_nothing_to_accept(store, where):
    """A plain step that fails has overwritten drafted tokens and advanced layers; one that is refused has not."""
    model = _cpu_model(store)
    with torch.no_grad():
        cache = model.new_cache(max_len=16, kv_bits=8)
        model(_ids(model, IDS[:5]), cache)
        model.verify(_ids(model, DRAFT), cache, PARENTS)
        with pytest.raises(ValueError, match="positions"):
            model(_ids(model, [1] * 12), cache)
        assert cache.drafted is not None
        if where == "replay":
            graph = object.__new__(GraphDecoder)
            graph.cache, graph.ids, graph.graph = cache, _ids(model, [0]), _Fails()
            step = graph.step
        else:
            step = lambda ids: model(ids, cache)  # noqa: E731
            if where == "head":
                model.lm_head = _Fails()
            else:
                model.layers[-1].down = _Fails()
        with pytest.raises(RuntimeError, match="memory"):
            step(_ids(model, [4]))
        with pytest.raises(ValueError, match="verify"):
            model.accept(cache, [1, 5])


def test_cpu_failed_accept_is_not_repeated(store, monkeypatch):
    """A layer's state that cannot be advanced: earlier layers have been, and K and V rows moved. A path that is
    refused changes nothing and may be followed by another."""
    model = _cpu_model(store)
    with torch.no_grad():
        cache = model.new_cache(max_len=16, kv_bits=8)
        model(_ids(model, IDS[:5]), cache)
        model.verify(_ids(model, DRAFT), cache, PARENTS)
        with pytest.raises(ValueError, match="path"):
            model.accept(cache, [5])
        assert cache.drafted is not None
        monkeypatch.setattr(model.layers[1].mixer, "advance", _Fails().forward)
        with pytest.raises(RuntimeError, match="memory"):
            model.accept(cache, [1, 5])
        monkeypatch.undo()
        with pytest.raises(ValueError, match="verify"):
            model.accept(cache, [1, 5])


def test_cpu_attention_layer_refuses_a_tree_on_a_16_bit_cache(store):
    """It would run as a sequence there."""
    layer, x = _cpu_model(store).layers[3].mixer, torch.randn(1, 3, ARGS.hidden_size)
    tree = torch.tensor([-1, 0, 0], dtype=torch.int32)
    with torch.no_grad():
        cache = Qwen35Cache(ARGS, 1, 8, "cpu", torch.float32)
        with pytest.raises(ValueError, match="8-bit"):
            layer(x, cache, parents=tree)
        assert not cache.k[3].any()
        layer(x, Qwen35Cache(ARGS, 1, 8, "cpu", torch.float32, kv_bits=8), parents=tree)


class _Returns(torch.nn.Module):
    def __init__(self, out):
        super().__init__()
        self.out = out

    def forward(self, x):
        return self.out


@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("parents", [None, [-1, 0, 0, 1, 1, -1]])
def test_cpu_rows_that_are_not_finite(parents, name):
    """A new token's K or V row with a NaN or an infinity reaches the tokens that see it, in its KV head's query heads,
    and no other."""
    from mlx_gsq_amd.models.qwen35 import FullAttention
    g = torch.Generator().manual_seed(7)
    a, B, S = ARGS, 2, 6
    H, G, hd = a.num_attention_heads, a.num_key_value_heads, a.head_dim
    rows = {"qk": torch.randn(B, S, H * 2 * hd + G * hd, generator=g), "v": torch.randn(B, S, G * hd, generator=g)}
    tree = None if parents is None else torch.tensor(parents, dtype=torch.int32)

    def run(qk, v):
        m = FullAttention(a, 3, _Returns(qk), _Returns(v), torch.nn.Identity(), torch.ones(hd), torch.ones(hd))
        with torch.no_grad():
            return m(torch.zeros(B, S, 8), Qwen35Cache(a, B, 16, "cpu", torch.float32, kv_bits=8), parents=tree).view(B, S, H, hd)
    clean = run(**rows)
    assert torch.isfinite(clean).all()
    for node, value in ((5, float("nan")), (1, float("inf"))):
        bad = {n: t.clone() for n, t in rows.items()}
        if name == "k":
            bad["qk"][1, node, H * 2 * hd + (G - 1) * hd + 3] = value
        else:
            bad["v"][1, node, (G - 1) * hd + 3] = value
        got = run(**bad)
        sees = [node <= t if parents is None else _on_path(parents, node, t) for t in range(S)]
        hit = torch.zeros(B, S, H, hd, dtype=torch.bool)
        hit[1, sees, H - H // G:] = True
        assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])


def _on_path(parents, node, t):
    while t > node:
        t = parents[t]
    return t == node


@pytest.mark.gpu
def test_gpu_8_bit_cache_and_tree():
    """Against the CPU's float32 model within the bound of the fp16 decoder (2e-2), and among themselves: trees
    against single tokens, prompts against single tokens, graph replays against eager steps."""
    model = _gpu_model()
    cpu = _cpu_model(TinyStore("cpu", seed=1))
    with torch.no_grad():
        want = cpu(_ids(cpu, IDS), cpu.new_cache(max_len=16, kv_bits=8))
        pre = model(_ids(model, IDS), model.new_cache(max_len=32, kv_bits=8))
        dec = _one_at_a_time(model, IDS)
        assert rel_l2(pre.float().cpu().numpy(), want.numpy()) <= 2e-2
        assert rel_l2(dec.float().cpu().numpy(), want.numpy()) <= 2e-2
        _check_tree(model, 2e-2)
        cache = model.new_cache(max_len=32, kv_bits=8)
        graph = GraphDecoder(model, cache)
        for i, t in enumerate(IDS):
            assert torch.equal(graph.step(_ids(model, [t]))[:, 0], dec[:, i]), i
        # a tree behind replayed steps
        logits = model.verify(_ids(model, DRAFT), cache, PARENTS)
        model.accept(cache, [0, 2])
        step = graph.step(_ids(model, [77]))[:, 0].clone()
        seq = _one_at_a_time(model, IDS + [DRAFT[0], DRAFT[2], 77])
        assert rel_l2(logits[:, 2].float().cpu().numpy(), seq[:, -2].float().cpu().numpy()) <= 2e-2
        assert rel_l2(step.float().cpu().numpy(), seq[:, -1].float().cpu().numpy()) <= 2e-2
        # a replayed step forgets the drafted tokens
        model.verify(_ids(model, DRAFT), cache, PARENTS)
        graph.step(_ids(model, [5]))
        with pytest.raises(ValueError, match="verify"):
            model.accept(cache, [0])
        # single drafted token: the cache stays as it was
        cache2 = model.new_cache(max_len=32, kv_bits=8)
        model(_ids(model, IDS), cache2)
        kept = [t.clone() for t in (*cache2.rec.values(), *cache2.conv.values())]
        one = model.verify(_ids(model, [9]), cache2, [-1])
        assert all(torch.equal(a, b) for a, b in zip(kept, (*cache2.rec.values(), *cache2.conv.values())))
        assert rel_l2(one[:, 0].float().cpu().numpy(), _one_at_a_time(model, IDS + [9])[:, -1].float().cpu().numpy()) <= 2e-2
        # parents on the device that are none: NaN, not a fault
        bad = model.verify(_ids(model, DRAFT), cache2, torch.tensor([-1, 1, 0, 2, 2, 1, 3], device="cuda"))
        assert torch.isnan(bad).all()


@pytest.mark.gpu
def test_gpu_float32_activations_take_the_torch_formulation():
    """The kernels serve 16-bit activations; others run the same definition in torch ops on the GPU."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mlx_gsq_amd.models.qwen35 import FullAttention
    g = torch.Generator().manual_seed(3)
    a = ARGS
    H, G, hd = a.num_attention_heads, a.num_key_value_heads, a.head_dim
    rows = torch.randn(1, 6, H * 2 * hd + G * hd, generator=g), torch.randn(1, 6, G * hd, generator=g)

    class Given(torch.nn.Module):
        def __init__(self, v):
            super().__init__()
            self.v = v

        def forward(self, x):
            return self.v
    outs = []
    for dev in ("cpu", "cuda"):
        qk, v = (t.to(dev) for t in rows)
        m = FullAttention(a, 3, Given(qk), Given(v), torch.nn.Identity(), torch.ones(hd, device=dev), torch.ones(hd, device=dev))
        cache = Qwen35Cache(a, 1, 16, dev, torch.float32, kv_bits=8)
        parents = torch.tensor([-1, 0, 0, 1, 1, -1], dtype=torch.int32, device=dev)
        outs.append(m(torch.zeros(1, 6, 8, device=dev), cache, parents=parents).cpu())
    assert rel_l2(outs[1].numpy(), outs[0].numpy()) <= 1e-5
