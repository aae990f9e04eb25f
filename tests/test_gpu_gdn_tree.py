"""GatedDeltaNet over a tree of drafted tokens (``gdn_tree``) against a float64 recurrence along every path:
tree sizes around the 16-row tiles, every kind of tree, head dims, convolution kernels and activation
types; against ``gdn_seq`` on a path; values that are not finite and parents that are none."""
import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# (batch, tokens, key heads, value heads, key dim, value dim, convolution kernel, row padding, dtype, tree)
CASES = [(1, 1, 2, 2, 128, 64, 4, 0, F16, "random"), (2, 2, 2, 6, 128, 128, 4, 0, F16, "star"),
         (1, 15, 3, 3, 64, 64, 2, 0, F16, "random"), (3, 16, 1, 2, 32, 192, 4, 0, BF16, "random"),
         (2, 17, 2, 4, 128, 128, 8, 3, F16, "chain"), (1, 33, 3, 3, 32, 256, 3, 1, F32, "random"),
         (1, 48, 8, 16, 64, 128, 4, 3, F32, "random"), (2, 64, 2, 6, 128, 128, 4, 0, F16, "random"),
         (1, 64, 1, 1, 128, 256, 4, 0, BF16, "chain"), (1, 64, 16, 48, 128, 128, 4, 0, BF16, "star"),
         (1, 9, 2, 4, 96, 64, 4, 0, F16, "random"), (2, 31, 2, 2, 4, 64, 5, 0, F32, "chain"),
         (1, 32, 1, 3, 100, 128, 4, 0, F32, "random")]


def _inputs(case, seed=0):
    B, S, hk, hv, dk, dv, K, pad, dtype, tree = case
    g = torch.Generator().manual_seed(seed + 100 * S + dk)
    C = 2 * hk * dk + hv * dv

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(dtype)
    rows = rnd(B, S, C + hv * dv + pad)
    if tree == "chain":
        p = torch.arange(S).expand(B, S) - 1
    elif tree == "star":
        p = torch.full((B, S), -1)
    else:
        p = (torch.arange(S) - 1 - (torch.rand(B, S, generator=g) * 5).long()).clamp(min=-1)
    return {"rows": rows, "ab": rnd(B, S, 2 * hv), "conv": rnd(B, K - 1, C), "cw": 0.5 * rnd(C, K),
            "ssm_a": -torch.exp(2 * torch.rand(hv, generator=g)), "dt": torch.randn(hv, generator=g) - 2,
            "rec": torch.randn(B, hv, dk, dv, generator=g), "nw": 1 + 0.1 * rnd(dv), "parents": p.to(torch.int32).contiguous()}


def _run(case, t, op="gdn_tree"):
    from mlx_gsq_amd.runtime.kernels import model_ops
    B, S, hk, hv, dk, dv, K, pad, dtype, tree = case
    d = {n: x.cuda() for n, x in t.items()}
    C = 2 * hk * dk + hv * dv
    args = [d["rows"][..., :C], d["rows"][..., C:C + hv * dv], d["ab"], d["conv"], d["cw"], d["ssm_a"], d["dt"], d["rec"], d["nw"]]
    kw = dict(key_heads=hk, value_heads=hv, head_k_dim=dk, head_v_dim=dv, eps=1e-6)
    if op == "gdn_tree":
        out = model_ops.gdn_tree(*args, d["parents"], **kw)
        assert torch.equal(d["rec"].cpu(), t["rec"]) and torch.equal(d["conv"].cpu(), t["conv"])
    else:
        out = model_ops.gdn_seq(*args, **kw)
    return out.cpu()


def _reference(case, t):
    """float64, each token from its parent's state and window."""
    B, S, hk, hv, dk, dv, K, pad, dtype, tree = case
    C = 2 * hk * dk + hv * dv
    x, head = t["rows"].double(), torch.arange(hv) % hk
    out = torch.empty(B, S, hv, dv, dtype=torch.float64)

    def norm(v, e):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + e)
    for b in range(B):
        states, windows = {-1: t["rec"][b].double()}, {-1: t["conv"][b].double()}
        for i in range(S):
            p = int(t["parents"].expand(B, S)[b, i])
            win = torch.cat([windows[p], x[b, i:i + 1, :C]])
            windows[i] = win[1:]
            y = (win * t["cw"].double().t()).sum(0)
            q, k, v = (y * torch.sigmoid(y)).split([hk * dk, hk * dk, hv * dv])
            q, k = (norm(q.view(hk, dk), 1e-6) / dk)[head], (norm(k.view(hk, dk), 1e-6) * dk ** -0.5)[head]
            a, beta = t["ab"][b, i].double().split(hv)
            decay = torch.exp(t["ssm_a"].double() * torch.nn.functional.softplus(a + t["dt"].double()))
            st = states[p] * decay[:, None, None]
            delta = (v.view(hv, dv) - (st * k[..., None]).sum(1)) * torch.sigmoid(beta)[:, None]
            states[i] = st + k[..., None] * delta[:, None]
            out[b, i] = (states[i] * q[..., None]).sum(1)
    z = x[..., C:C + hv * dv].reshape(B, S, hv, dv)
    return (norm(out, 1e-6) * t["nw"].double() * z * torch.sigmoid(z)).reshape(B, S, hv * dv)


def _bound(dtype):
    """rel-L2: one rounding of the outputs, and float32 sums: four stages (norms, scores, system, outputs) of
    up to 128 + 64 terms in steps of 4, whose terms are up to sqrt(128) times the sum: 4 x 48 x 11 x 2^-24 at most."""
    return (0.0 if dtype == F32 else torch.finfo(dtype).eps / 2) + 4 * 48 * 11 * 2.0 ** -24


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
def test_gdn_tree_matches_float64(case):
    t = _inputs(case)
    got, want = _run(case, t), _reference(case, t)
    assert torch.isfinite(got).all()
    assert _rel(got, want) <= _bound(case[8])
    shared = dict(t, parents=t["parents"][0].contiguous())  # one tree for all batch rows
    assert _rel(_run(case, shared), _reference(case, shared)) <= _bound(case[8])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_gdn_tree_chain_is_gdn_seq(dtype):
    """A tree that is a sequence: gdn_seq's outputs, whose float32 sums go in another order."""
    case = (2, 40, 2, 6, 128, 128, 4, 0, dtype, "chain")
    t = _inputs(case, 3)
    assert _rel(_run(case, t), _run(case, t, "gdn_seq")) <= 2 * _bound(dtype)


def test_gdn_tree_repeated_tokens_and_strong_decays():
    """Keys that are all alike (the system's weights are beta everywhere) with beta near 1, and decays from
    e^-40 to 1 on one path, behind which ratios stay exact."""
    case = (1, 64, 1, 2, 64, 64, 4, 0, F32, "chain")
    t = _inputs(case, 5)
    t["rows"][:, :, :2 * 64] = t["rows"][:, :1, :2 * 64]
    t["conv"][:] = t["rows"][:, :1, :2 * 64 + 128]
    t["ab"][..., 2:] = 6.0
    t["ab"][..., :2] = -8.0
    t["ab"][:, 5::16, :2] = 40.0
    t["ssm_a"][:] = -1.0
    # the weights' inverse has entries up to 64 in size sums of 64 of them: 16 times the bound's cancellation
    assert _rel(_run(case, t), _reference(case, t)) <= 16 * _bound(F32)


def test_gdn_tree_not_finite():
    """A NaN in a token's inputs or gates reaches the tokens behind it, in the heads that read it, and no other."""
    case = (2, 37, 2, 4, 64, 64, 4, 0, F16, "random")
    B, S, hk, hv, dk, dv, K, pad, dtype, tree = case
    t = _inputs(case, 7)
    clean = _run(case, t).view(B, S, hv, dv)
    C = 2 * hk * dk + hv * dv
    node = 4

    def below(b, steps=99):  # tokens within that many steps behind the node, itself among them
        out = []
        for i in range(S):
            j, n = i, 0
            while j > node and n < steps:
                j, n = int(t["parents"][b, j]), n + 1
            out.append(j == node)
        return out

    def check(name, at, value, steps, heads):
        x = t[name].clone()
        x[at] = value
        got = _run(case, dict(t, **{name: x})).view(B, S, hv, dv)
        bad = torch.zeros(B, S, hv, dv, dtype=torch.bool)
        for h in heads:
            bad[1, below(1, steps), h] = True
        assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])
    nan = float("nan")
    check("rows", (1, node, 64 + 3), nan, K - 1, (1, 3))             # q of key head 1: the windows that hold it
    check("rows", (1, node, 2 * 64 + 5), nan, 99, (0, 2))            # k of key head 0
    check("rows", (1, node, 4 * 64 + 2 * 64 + 9), nan, 99, (2,))     # v of value head 2
    check("ab", (1, node, 1), nan, 99, (1,))                         # decay of head 1
    check("ab", (1, node, hv + 3), nan, 99, (3,))                    # beta of head 3
    x = t["rows"].clone()
    x[1, node, C + 7] = nan                                          # its output gate: its value alone
    got = _run(case, dict(t, rows=x)).view(B, S, hv, dv)
    assert torch.isnan(got[1, node, 0, 7])
    got[1, node, 0, 7] = clean[1, node, 0, 7]
    assert torch.equal(got, clean)


def test_gdn_tree_bad_parents():
    case = (3, 20, 1, 2, 32, 64, 4, 0, F16, "random")
    t = _inputs(case, 9)
    clean = _run(case, t)
    for i, p in ((0, 0), (5, 5), (5, 19), (3, -2), (19, 2 ** 30)):
        bad = t["parents"].clone()
        bad[1, i] = p
        got = _run(case, dict(t, parents=bad))
        assert torch.isnan(got[1]).all() and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


def test_gdn_tree_graph_replays():
    from mlx_gsq_amd.runtime.kernels import model_ops
    case = (2, 21, 2, 6, 128, 128, 4, 0, F16, "random")
    B, S, hk, hv, dk, dv, K, pad, dtype, tree = case
    d = {n: x.cuda() for n, x in _inputs(case, 11).items()}
    C = 2 * hk * dk + hv * dv

    def call():
        return model_ops.gdn_tree(d["rows"][..., :C], d["rows"][..., C:], d["ab"], d["conv"], d["cw"], d["ssm_a"], d["dt"],
                                  d["rec"], d["nw"], d["parents"], key_heads=hk, value_heads=hv, head_k_dim=dk, head_v_dim=dv,
                                  eps=1e-6)
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for i in range(3):
        want = call()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        d["rows"].mul_(0.9)
        d["rec"].mul_(1.1)
        d["parents"][:, 1:].clamp_(max=i)


@pytest.mark.parametrize("a", [3e4, 1e18, float("inf")])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gdn_tree_decays_of_nothing(dtype, a):
    """Tokens that forget everything before them (decays of e^-3e4 and less): the decays of those that follow keep
    their bits."""
    case = (1, 40, 2, 4, 64, 64, 4, 0, dtype, "random")
    t = _inputs(case, 13)
    t["ab"][:, 3::9, :4] = a
    want = _reference(case, t)
    assert torch.isfinite(want).all()
    assert _rel(_run(case, t), want) <= _bound(dtype)
    chain = dict(t, parents=(torch.arange(40, dtype=torch.int32) - 1)[None].contiguous())
    want = _reference(case, chain)
    assert _rel(_run(case, chain), want) <= _bound(dtype) and _rel(_run(case, chain, "gdn_seq"), want) <= _bound(dtype)


@pytest.mark.parametrize("size", [1e-5, 1e-7])
def test_gdn_tree_small_queries_and_keys(size):
    """q and k inputs far below the norm's epsilon (their rows are 1000 times the inputs, not of size 1): float32's bits
    all the same."""
    case = (1, 20, 2, 4, 128, 64, 4, 0, F32, "random")
    t = _inputs(case, 17)
    n = 2 * 2 * 128
    t["rows"][..., :n] *= size
    t["conv"][..., :n] *= size
    assert _rel(_run(case, t), _reference(case, t)) <= _bound(F32)
