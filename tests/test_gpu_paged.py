"""Steps of packed requests over paged caches (``page_plan``, ``paged_write``, ``attn_paged``, ``gdn_packed``) against
their definitions: whole numbers exactly, the rest in float64."""
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

F16, BF16 = torch.float16, torch.bfloat16


def _paged():
    from mlx_gsq_amd.runtime.kernels import paged
    return paged


def _name(c):
    return "-".join(map(str, c)).replace("torch.", "").replace(" ", "")


# ---- plans ---------------------------------------------------------------------------------------

# (requests, new tokens, lengths, pages held, table width, free pages, rows, page size)
PLANS = [([0], [1], [0], [0], 1, 1, 1, 16),
         ([2, 0, 1], [1, 1, 1], [15, 16, 0], [1, 1, 0], 4, 5, 3, 16),
         ([1, 0], [40, 1], [0, 31, 7], [0, 1, 1], 3, 9, 50, 32),            # rows behind the last sequence
         ([3, 1, 0, 2], [100, 20, 1, 0], [0, 12, 64, 5], [0, 1, 1, 1], 8, 3, 200, 64),  # pages run out, need of none is served
         ([0, 0, 5, -1, 1], [4, 4, 1, 1, 2], [3, 3], [1, 1], 2, 4, 12, 16),  # named twice, out of range
         ([0, 1], [30, 3], [0, 0], [0, 0], 1, 5, 33, 16),                    # longer than a table row
         ([0, 1, 2], [5, 8, 3], [0, 0, 0], [0, 0, 0], 2, 9, 10, 16),         # more tokens than rows
         ([0, 1], [-2, 3], [4, 4], [1, 1], 2, 2, 5, 16),                     # fewer than no tokens
         ([1, 0], [1, 1], [10, 3], [4, 2], 5, 0, 2, 16),                     # more pages held than needed
         ([], [], [3, 4], [1, 1], 2, 2, 4, 16)]


def _plan_state(case, g):
    requests, new, lengths, held, W, spare, tokens, page = case
    order = torch.randperm(sum(held) + spare + 3, generator=g).tolist()
    table = [[-1] * W for _ in lengths]
    for r, h in enumerate(held):
        table[r][:h] = [order.pop() for _ in range(h)]
    free = [order.pop() for _ in range(spare)]
    return requests, new, list(lengths), list(held), table, free + [-1] * (sum(held) + 3), spare, tokens, page


def _on_gpu(requests, new, lengths, held, table, free, n_free):
    return [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (requests, new, lengths, held, table, free, [n_free])]


@pytest.mark.parametrize("case", PLANS, ids=range(len(PLANS)))
def test_page_plan_matches_definition(case):
    requests, new, lengths, held, table, free, n_free, tokens, page = _plan_state(case, R.gen(case))
    d = _on_gpu(requests, new, lengths, held, table, free, n_free)
    for _ in range(2):  # the second call finds the pages held
        got = _paged().page_plan(*d, tokens=tokens, page_size=page)
        want, n_free = R.plan(requests, new, lengths, held, table, free, n_free, tokens, page)
        for name, x, y in zip(got._fields, got, want):
            assert x.tolist() == y, name
        assert d[3].tolist() == held and d[4].tolist() == table and d[5].tolist() == free and d[6].tolist() == [n_free]
        assert d[2].tolist() == lengths
    _paged().page_advance(got, d[2])
    for r, n in zip(want[1], want[2]):
        if r >= 0:
            lengths[r] = n
    assert d[2].tolist() == lengths


@pytest.mark.parametrize("B", [1, 63, 64, 65, 300, 1024])
def test_page_plan_of_many_sequences(B):
    g = R.gen("many", B)
    page, Rn = 16, B + 3
    requests = torch.randperm(Rn, generator=g)[:B].tolist()
    lengths = torch.randint(0, 200, (Rn,), generator=g).tolist()
    held = [-(-n // page) for n in lengths]
    new = (torch.randint(0, 40, (B,), generator=g) * (torch.rand(B, generator=g) < 0.4)).tolist()
    case = (requests, new, lengths, held, 16, sum(new) // page + B // 2, sum(new) + 7, page)
    requests, new, lengths, held, table, free, n_free, tokens, page = _plan_state(case, g)
    first = [list(free), n_free, [list(x) for x in table], list(held), list(lengths)]
    d = _on_gpu(requests, new, lengths, held, table, free, n_free)
    got = _paged().page_plan(*d, tokens=tokens, page_size=page)
    want, n_free = R.plan(requests, new, lengths, held, table, free, n_free, tokens, page)
    for name, x, y in zip(got._fields, got, want):
        assert x.tolist() == y, name
    assert d[4].tolist() == table and d[6].tolist() == [n_free]
    # back they go, some named twice or out of range
    back = requests[: B // 2 + 1] + [requests[0], -7, Rn]
    back = back[:1024]
    _paged().page_release(torch.tensor(back, dtype=torch.int32, device="cuda"), d[2], d[3], d[4], d[5], d[6])
    n_free = R.release(back, lengths, held, table, free, n_free)
    assert d[6].tolist() == [n_free] and d[5].tolist()[:n_free] == free[:n_free]
    assert d[2].tolist() == lengths and d[3].tolist() == held and d[4].tolist() == table
    del first


def test_release_gives_back_what_a_plan_took():
    case = ([2, 0, 1], [70, 33, 5], [0, 0, 0], [0, 0, 0], 8, 20, 120, 16)
    requests, new, lengths, held, table, free, n_free, tokens, page = _plan_state(case, R.gen("back"))
    d = _on_gpu(requests, new, lengths, held, table, free, n_free)
    before = [x.clone() for x in d]
    _paged().page_plan(*d, tokens=tokens, page_size=page)
    assert int(d[6]) < n_free
    _paged().page_release(d[0], *d[2:])
    assert all(torch.equal(x, y) for x, y in zip(before, d))


# ---- writing -------------------------------------------------------------------------------------

# (cached, new, page, heads, kv heads, head dim, rotary dim, dtype, element offset of the rows)
WRITES = [([0], [1], 16, 1, 1, 64, 0, F16, 0), ([5, 511], [1, 1], 64, 24, 4, 256, 64, BF16, 0),
          ([0, 9, 4], [7, 1, 30], 16, 6, 2, 128, 128, F16, 0), ([40], [33], 32, 4, 4, 64, 6, BF16, 0),
          ([70001, 3], [300, 5], 256, 12, 2, 256, 64, F16, 1), ([0], [1500], 128, 5, 1, 128, 32, BF16, 0),
          ([1000, 0, 0], [1, 0, 17], 16, 8, 8, 256, 256, F16, 0), ([2000000000], [3], 64, 3, 1, 64, 64, F16, 3),
          ([7], [1030], 64, 24, 4, 256, 64, BF16, 8)]


@pytest.mark.parametrize("case", WRITES, ids=_name)
def test_paged_write_matches_definition(case):
    cached, new, page, H, G, hd, rd, dtype, shift = case
    g = R.gen(case)
    far = max(cached) > 1 << 20  # a few pages stand for many
    table, plan, n_pages = R.step([c % page for c in cached] if far else cached, new, page, g, tail=2)
    pos = plan[3].clone()
    if far:
        pos[pos >= 0] += cached[0] - cached[0] % page
    N = pos.numel()

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(dtype)
    width = shift + H * 2 * hd + 2 * G * hd + 2 * (shift > 0)
    rows = rnd(N, width)  # [q | gate] of each head, k, v: one product's rows
    qw, kw = 1 + 0.2 * rnd(hd), 1 + 0.2 * rnd(hd)
    freq = 1e7 ** (-torch.arange(0, rd, 2).double() / max(rd, 1))
    kp, vp = rnd(n_pages, G, page, hd), rnd(n_pages, G, page, hd)

    def parts(r):
        n = shift + H * 2 * hd
        return r[:, shift:n].view(N, H, 2 * hd)[..., :hd], r[:, n:n + G * hd].view(N, G, hd), r[:, n + G * hd:n + 2 * G * hd].view(N, G, hd)
    dev = [x.cuda() for x in (qw, kw, freq, kp, vp, pos, plan[4])]
    got = _paged().paged_write(*parts(rows.cuda()), *dev, eps=1e-6).cpu()
    q, k, v = parts(rows)

    def turned(x, w):
        x = x.double()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        ang = pos.double()[:, None, None] * freq
        lo, hi = x[..., :rd // 2], x[..., rd // 2:rd]
        return torch.cat([lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin(), x[..., rd:]], -1)
    # one rounding to dtype; norm, rotation and its factors in float32: 16 roundings of the row's size, and 2^-21 of
    # it twice for a sine and a cosine that are 2^-22.3 (the reduced angle) + 2^-23 off; turns in double at far positions
    eps = torch.finfo(dtype).eps / 2
    turn = float(pos.max()) * 2.0 ** -51

    def close(x, want):
        err = (x.double() - want).abs()
        top = want.abs().amax(-1, keepdim=True) * (2 ** 0.5 if rd else 1)
        assert bool((err <= eps * want.abs() + (2.0 ** -20 + 2.0 ** -20 + 2 * turn) * (1 + eps) * top + 2.0 ** -25).all()), float(err.max())
    there = plan[4] >= 0
    close(got[there], turned(q, qw)[there])
    assert not bool(got[~there].any())
    want_k, want_v, at = kp.clone(), vp.clone(), plan[4][there]
    got_k, got_v = dev[3].cpu(), dev[4].cpu()
    close(got_k[at // page, :, at % page], turned(k, kw)[there])
    want_k[at // page, :, at % page] = got_k[at // page, :, at % page]
    want_v[at // page, :, at % page] = v[there]
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)  # nothing else is touched


# ---- attention -----------------------------------------------------------------------------------

def _attn_inputs(cached, new, page, H, G, hd, dtype, key, tail=0, k_size=1.0):
    g = R.gen(key)
    table, plan, n_pages = R.step(cached, new, page, g, tail=tail)
    N = plan[3].numel()
    q = torch.randn(N, H, hd, generator=g).to(dtype)
    kp = (k_size * torch.randn(n_pages, G, page, hd, generator=g)).to(dtype)
    vp = (torch.randn(n_pages, G, page, hd, generator=g) * torch.exp(0.5 * torch.randn(n_pages, G, page, 1, generator=g))).to(dtype)
    gate = torch.randn(N, H, 2 * hd, generator=g).to(dtype)
    return q, kp, vp, table, plan, gate


def _attend(q, kp, vp, table, plan, gate=None, **kw):
    P = _paged()
    return P.attn_paged(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), P.PagePlan(*(x.cuda() for x in plan)),
                        gate=None if gate is None else gate.cuda()[..., gate.shape[-1] // 2:], **kw).cpu()


def _check_attn(got, q, kp, vp, table, plan, gate):
    half = None if gate is None else gate[..., gate.shape[-1] // 2:]
    want, size, score = R.attention(q, kp, vp, table, *plan[:3], half)
    err = (got.double() - want).abs()
    bound = R.attention_bound(want, size, score, q.dtype, q.shape[2], int(plan[2].max()) if len(plan[2]) else 0)
    assert bool((err <= bound).all()), float((err - bound).max())
    if float(want.norm()):
        assert float((got.double() - want).norm() / want.norm()) <= torch.finfo(q.dtype).eps / 2 + 1e-4


# (cached, new, page, heads, kv heads, head dim, dtype)
ATTNS = [([0], [1], 16, 1, 1, 64, F16), ([300], [1], 16, 24, 4, 256, F16), ([0, 15, 16, 17, 31, 32, 33, 63, 64, 65], [1] * 10, 16, 6, 1, 256, BF16),
         ([5000, 0, 77, 1300], [1, 1, 1, 1], 64, 8, 2, 128, BF16), ([3000, 255, 256, 257], [1] * 4, 256, 16, 4, 64, F16),
         ([0], [2], 32, 24, 4, 256, BF16), ([0], [333], 64, 6, 1, 256, F16), ([0, 0, 0], [65, 1, 130], 16, 8, 2, 128, BF16),
         ([100, 0, 31], [17, 0, 40], 16, 4, 4, 64, F16), ([1000, 500, 7, 0], [50, 1, 1, 129], 128, 12, 2, 256, BF16),
         ([640], [200], 16, 5, 1, 128, F16), ([2100, 9], [70, 1], 32, 64, 8, 64, BF16), ([9000], [33], 64, 2, 1, 256, F16),
         ([0], [700], 64, 8, 1, 64, BF16), ([20, 4], [3, 5], 16, 40, 8, 128, F16)]


@pytest.mark.parametrize("case", ATTNS, ids=_name)
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
def test_attn_paged_matches_definition(case, gated):
    q, kp, vp, table, plan, gate = _attn_inputs(*case, key=case, tail=3)
    gate = gate if gated else None
    for hint in ({}, {"max_new": max(case[1])}):
        got = _attend(q, kp, vp, table, plan, gate, **hint)
        _check_attn(got[:-3], q[:-3], kp, vp, table, plan, None if gate is None else gate[:-3])
        assert not bool(got[-3:].any())  # behind the last sequence


def test_attn_paged_follows_no_hint():
    """Sequences of more new tokens than max_new says are served too."""
    case = ([0, 40], [150, 90], 16, 6, 2, 128, F16)
    q, kp, vp, table, plan, gate = _attn_inputs(*case, key="hint")
    for most in (1, 5, 1000):
        _check_attn(_attend(q, kp, vp, table, plan, gate, max_new=most), q, kp, vp, table, plan, gate)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_attn_paged_wide_scores(hd, dtype):
    """Scores from one weight of nearly 1 to ranges past what a weight can hold, at every split and tile."""
    for k_size in (0.01, 6.0, 60.0):
        q, kp, vp, table, plan, gate = _attn_inputs([900, 0, 3000], [1, 140, 2], 32, 4, 2, hd, dtype, key=(hd, k_size), k_size=k_size)
        _check_attn(_attend(q, kp, vp, table, plan, gate), q, kp, vp, table, plan, gate)


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attn_paged_masked_places_do_not_reach(hd, value):
    """K and V rows that a token does not see, of whatever values, leave its outputs alone: later tokens of its own prompt,
    the rest of a page, pages of others."""
    cached, new = [37, 0, 5], [1, 90, 20]
    q, kp, vp, table, plan, gate = _attn_inputs(cached, new, 16, 6, 2, hd, F16, key=("masked", hd), tail=1)
    cu, rows, lens = (x.tolist() for x in plan[:3])
    used = torch.zeros(kp.shape[0], 16, dtype=torch.bool)
    for r, n in zip(rows, lens):
        for p in range(n):
            used[table[r, p // 16], p % 16] = True
    for c in (kp, vp):
        c.transpose(1, 2)[~used] = value
    for b, at in ((1, 60), (2, 19)):  # token `at` of sequence b: the tokens before it do not see it
        p = lens[b] - new[b] + at
        vp[table[rows[b], p // 16], :, p % 16] = value
        kp[table[rows[b], p // 16], :, p % 16, 3] = value
    got = _attend(q, kp, vp, table, plan, gate)
    free = torch.ones(q.shape[0], dtype=torch.bool)
    free[cu[1] + 60:cu[2]] = False
    free[cu[2] + 19] = False
    free[-1] = False
    want, size, score = R.attention(q, kp.nan_to_num(0, 0, 0), vp.nan_to_num(0, 0, 0), table, *plan[:3], gate[..., hd:])
    bound = R.attention_bound(want, size, score, F16, hd, 110)
    assert bool(((got.double() - want).abs() <= bound)[free].all())


def test_attn_paged_visible_infinities():
    """A visible V of infinity is an output of infinity (or NaN where its weight is 0), a visible NaN key one of NaN."""
    q, kp, vp, table, plan, gate = _attn_inputs([0, 50], [40, 1], 16, 4, 1, 64, BF16, key="visible", k_size=0.1)
    rows = plan[1].tolist()
    vp[table[rows[0], 0], 0, 7, 5] = float("inf")       # position 7 of the prompt, dim 5
    kp[table[rows[1], 1], 0, 2, 0] = float("nan")       # position 18 of the other request
    got = _attend(q, kp, vp, table, plan)
    assert bool(torch.isfinite(got[:7]).all()) and bool(torch.isinf(got[7:40, :, 5]).all())
    keep = torch.arange(64) != 5
    assert bool(torch.isfinite(got[:40][..., keep]).all()) and bool(torch.isnan(got[40]).all())


def test_attn_paged_rows_not_served():
    """Sequences that are not served, or whose numbers do not fit, are NaN; the others are as they were."""
    case = ([10, 40, 3, 20], [2, 30, 1, 5], 16, 6, 2, 128, F16)
    q, kp, vp, table, plan, gate = _attn_inputs(*case, key="served")
    want = _attend(q, kp, vp, table, plan, gate)
    cu, rows, lens = plan[0].tolist(), plan[1].tolist(), plan[2].tolist()
    for b, change in ((0, ("rows", -1)), (1, ("rows", table.shape[0])), (1, ("lens", 29)), (2, ("lens", 1 << 30)),
                      (3, ("page", -1)), (1, ("page", kp.shape[0])), (3, ("page", 1 << 30))):
        t, p = table.clone(), [x.clone() for x in plan]
        if change[0] == "page":
            t[rows[b], 1] = change[1]
        else:
            p[1 if change[0] == "rows" else 2][b] = change[1]
        got = _attend(q, kp, vp, t, p, gate)
        mine = torch.zeros(q.shape[0], dtype=torch.bool)
        mine[cu[b]:cu[b + 1]] = True
        assert bool(torch.isnan(got[mine]).all()), change
        assert torch.equal(got[~mine], want[~mine]), change


def test_attn_paged_repeats_exactly_on_streams_and_in_graphs():
    """The same inputs give the same bits: again, on another stream, and in a graph whose plan changes between replays."""
    P = _paged()
    case = ([700, 30, 0], [1, 1, 64], 16, 24, 4, 256, BF16)
    q, kp, vp, table, plan, gate = _attn_inputs(*case, key="graph")
    d = [x.cuda() for x in (q, kp, vp, table)]
    pl, gt = P.PagePlan(*(x.cuda() for x in plan)), gate.cuda()[..., 256:]
    want = P.attn_paged(*d, pl, gate=gt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = P.attn_paged(*d, pl, gate=gt)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = P.attn_paged(*d, pl, gate=gt)
    torch.cuda.synchronize()
    assert torch.equal(want, again)
    short = pl.lens.clone()
    short[0] = 300
    for i in range(4):
        pl.lens.copy_(short if i % 2 else plan[2].cuda())
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, P.attn_paged(*d, pl, gate=gt)), i
        assert torch.equal(got, want) == (i % 2 == 0)


# ---- GatedDeltaNet -------------------------------------------------------------------------------

# (cached, new, key heads, value heads, dk, dv, conv kernel, dtype)
GDNS = [([0], [1], 1, 1, 32, 64, 2, F16), ([3, 0, 900], [1, 1, 1], 16, 48, 128, 128, 4, BF16), ([0], [15], 2, 4, 64, 128, 4, F16),
        ([5, 0, 7, 1], [2, 17, 0, 64], 2, 2, 128, 64, 4, BF16), ([0, 11], [65, 130], 2, 6, 128, 128, 4, F16),
        ([100], [300], 1, 3, 128, 128, 4, BF16), ([0, 40, 0], [129, 1, 63], 2, 4, 64, 64, 3, F16), ([0, 8], [20, 200], 1, 2, 32, 256, 8, F16),
        ([0, 9], [1, 2], 4, 8, 32, 64, 5, BF16), ([60, 0, 2], [64, 128, 63], 1, 1, 128, 256, 4, F16)]


def _gdn_inputs(case, tail=0):
    cached, new, hk, hv, dk, dv, K, dtype = case
    g = R.gen(case)
    _, plan, _ = R.step(cached, new, 64, g, tail=tail)
    N, Rn, conv_dim = plan[3].numel(), len(new) + 2, 2 * hk * dk + hv * dv

    def rnd(*shape):
        return torch.randn(*shape, generator=g)
    qkvz = rnd(N, conv_dim + hv * dv + 2).to(dtype)
    ab = rnd(N, 2 * hv).to(dtype)
    a_log = torch.exp(torch.rand(hv, generator=g) * 2.77)
    t = (qkvz[:, :conv_dim], qkvz[:, conv_dim:conv_dim + hv * dv], ab, rnd(Rn, K - 1, conv_dim).to(dtype),
         (0.5 * rnd(conv_dim, K)).to(dtype), -a_log, torch.log(torch.expm1(torch.exp(torch.rand(hv, generator=g) * 4.6 - 6.9))),
         0.3 * rnd(Rn, hv, dk, dv), (1 + 0.1 * rnd(dv)).to(dtype))
    return t, plan


def _run_gdn(case, t, plan, **kw):
    P = _paged()
    cached, new, hk, hv, dk, dv, K, dtype = case
    n = t[0].shape[1]
    rows = torch.cat([t[0], t[1], t[1][:, :2]], 1).cuda()
    d = [rows[:, :n], rows[:, n:n + hv * dv]] + [x.cuda().clone() for x in t[2:]]
    out = P.gdn_packed(*d, P.PagePlan(*(x.cuda() for x in plan)), key_heads=hk, value_heads=hv, head_k_dim=dk, head_v_dim=dv,
                       eps=1e-6, **kw)
    return out.cpu(), d[3].cpu(), d[7].cpu()


def _check_gdn(case, t, plan, got):
    cached, new, hk, hv, dk, dv, K, dtype = case
    out, conv, rec = got
    want, want_conv, want_rec, scale = R.gdn(*t, *plan[:3], hk, hv, dk, dv, 1e-6)
    assert torch.equal(conv.double(), want_conv)
    # states: n products of 2^-22 and better, each at most the state's size, behind one another
    n = max(new)
    top = want_rec.abs().amax((-1, -2), keepdim=True)
    assert bool(((rec.double() - want_rec).abs() <= (n + 16) * 2.0 ** -21 * (top + 1)).all())
    assert float((rec.double() - want_rec).norm() / want_rec.norm()) <= 2e-6
    # outputs: one rounding; 2^-12 of the gated norm's factor for rows whose sum is a few hundred times smaller than its terms
    eps = torch.finfo(dtype).eps / 2
    err = (out.double() - want).abs()
    assert bool((err <= eps * want.abs() + 2.0 ** -12 * scale * dv ** 0.5 + 2.0 ** -25).all()), float(err.max())
    assert float((out.double() - want).norm() / want.norm()) <= eps + 1e-5


@pytest.mark.parametrize("case", GDNS, ids=_name)
def test_gdn_packed_matches_definition(case):
    t, plan = _gdn_inputs(case, tail=3)
    for hint in ({}, {"max_new": max(case[1])}):
        out, conv, rec = _run_gdn(case, t, plan, **hint)
        assert not bool(out[-3:].any())
        _check_gdn(case, tuple(x[:-3] for x in t[:3]) + t[3:], plan, (out[:-3], conv, rec))


def test_gdn_packed_follows_no_hint():
    case = ([0, 11], [65, 130], 2, 6, 128, 128, 4, F16)
    t, plan = _gdn_inputs(case)
    for most in (1, 20, 1000):
        _check_gdn(case, t, plan, _run_gdn(case, t, plan, max_new=most))


def test_gdn_packed_pieces_of_a_prompt():
    """A prompt in pieces leaves the state that it leaves whole, within the states' bound."""
    case = ([0], [200], 2, 4, 128, 128, 4, F16)
    t, plan = _gdn_inputs(case)
    whole = _run_gdn(case, t, plan)
    conv, rec, outs, at = t[3].clone(), t[7].clone(), [], 0
    for n in (1, 2, 70, 64, 3, 60):
        p = [x.clone() for x in plan]
        p[0], p[2] = torch.tensor([0, n], dtype=torch.int32), torch.tensor([at + n], dtype=torch.int32)
        part = tuple(x[at:at + n] for x in t[:3]) + (conv, *t[4:7], rec, t[8])
        o, conv, rec = _run_gdn((case[0], [n]) + case[2:], part, p)
        outs.append(o)
        at += n
    assert at == 200 and torch.equal(conv, whole[1])
    assert float((rec - whole[2]).norm() / whole[2].norm()) <= 2e-6
    assert float((torch.cat(outs).double() - whole[0].double()).norm() / whole[0].double().norm()) <= 2 * 2.0 ** -11


@pytest.mark.parametrize("where", ["k", "v", "q", "decay"])
def test_gdn_packed_values_that_are_not_finite(where):
    """They reach their own token and what follows it in its request, as in the recurrence, and nothing else."""
    case = ([0, 9, 3], [150, 70, 2], 1, 2, 64, 64, 4, F16)
    t, plan = _gdn_inputs(case)
    at = 100  # of the first sequence
    if where == "decay":
        t[2][at, 1] = -float("inf")  # softplus 0: nothing is forgotten
        t[2][at + 30, 0] = float("inf")  # everything is
    else:
        t[0][at, {"q": 3, "k": 64 + 5, "v": 128 + 64 + 7}[where]] = float("nan") if where == "k" else float("inf")
    out, conv, rec = _run_gdn(case, t, plan)
    want, want_conv, want_rec, scale = R.gdn(*t, *plan[:3], 1, 2, 64, 64, 1e-6)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and bool(torch.isfinite(out[:at]).all())
    assert torch.equal(torch.isnan(rec), torch.isnan(want_rec))
    assert bool(torch.isfinite(out[150:]).all()) and (where == "decay") == bool(torch.isfinite(out).all())
    err, fine = (out.double() - want).abs(), torch.isfinite(want)
    assert bool((err <= 2.0 ** -11 * want.abs() + 2.0 ** -9 * scale + 2.0 ** -25)[fine].all())
    fine = torch.isfinite(want_rec)
    assert float((rec.double() - want_rec)[fine].norm() / want_rec[fine].norm()) <= 2e-6


@pytest.mark.parametrize("conv_kernel,new", [(4, 3), (8, 7), (8, 30)])
def test_gdn_packed_windows_read_the_state_before_the_step(conv_kernel, new):
    """All tokens whose window begins before the step see the convolution state that the step before left."""
    case = ([5] * 40, [new - i % 3 for i in range(40)], 4, 8, 128, 128, conv_kernel, F16)
    t, plan = _gdn_inputs(case)
    first = None
    for _ in range(6):
        got = _run_gdn(case, t, plan)
        if first is None:
            first = got
            _check_gdn(case, t, plan, got)
        assert all(torch.equal(x, y) for x, y in zip(got, first))


def test_gdn_packed_begins_from_zeros():
    """A request's first tokens do not see what its states held."""
    case = ([0, 5], [70, 3], 1, 2, 128, 128, 4, BF16)
    t, plan = _gdn_inputs(case)
    r = int(plan[1][0])
    t[3][r], t[7][r] = float("nan"), float("nan")
    _check_gdn(case, t, plan, _run_gdn(case, t, plan))


def test_gdn_packed_rows_not_served():
    case = ([9, 4, 0], [3, 80, 2], 1, 2, 64, 64, 4, F16)
    t, plan = _gdn_inputs(case)
    want = _run_gdn(case, t, plan)
    cu, rows = plan[0].tolist(), plan[1].tolist()
    for b, (which, value) in ((0, (1, -1)), (1, (1, len(rows) + 2)), (1, (2, 79)), (2, (2, 1))):
        p = [x.clone() for x in plan]
        p[which][b] = value
        out, conv, rec = _run_gdn(case, t, p)
        mine = torch.zeros(out.shape[0], dtype=torch.bool)
        mine[cu[b]:cu[b + 1]] = True
        assert bool(torch.isnan(out[mine]).all()) and torch.equal(out[~mine], want[0][~mine])
        for got, w, before in ((conv, want[1], t[3]), (rec, want[2], t[7])):
            assert torch.equal(got[rows[b]], before[rows[b]])
            others = [r for r in range(w.shape[0]) if r != rows[b]]
            assert torch.equal(got[others], w[others])


# ---- a run of them -------------------------------------------------------------------------------

def test_a_step_as_it_is_used():
    """Plan, write, attend, advance, over three steps of two requests: what one pass over each whole request gives."""
    P = _paged()
    H, G, hd, rd, page, dtype = 6, 2, 64, 32, 16, F16
    g = R.gen("run")
    total, pieces = [50, 23], [[30, 1, 19], [0, 22, 1]]
    qkv = [torch.randn(n, H + 2 * G, hd, generator=g).to(dtype).cuda() for n in total]
    w = torch.ones(hd, dtype=dtype, device="cuda")
    freq = (1e4 ** (-torch.arange(0, rd, 2).double() / rd)).cuda()
    n_pages = 8
    kp, vp = (torch.full((n_pages, G, page, hd), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    i32 = dict(dtype=torch.int32, device="cuda")
    lengths, held = torch.zeros(3, **i32), torch.zeros(3, **i32)
    table, free, n_free = torch.full((3, 4), -1, **i32), torch.arange(n_pages, **i32), torch.tensor([n_pages], **i32)
    requests, outs, at = torch.tensor([2, 0], **i32), [[], []], [0, 0]
    for i in range(3):
        new = [p[i] for p in pieces]
        plan = P.page_plan(requests, torch.tensor(new, **i32), lengths, held, table, free, n_free, tokens=sum(new) + 1, page_size=page)
        x = torch.cat([qkv[r][at[r]:at[r] + n] for r, n in enumerate(new)] + [qkv[0][:1]])
        q = P.paged_write(x[:, :H], x[:, H:H + G], x[:, H + G:], w, w, freq, kp, vp, plan.pos, plan.slots, eps=1e-6)
        o = P.attn_paged(q, kp, vp, table, plan)
        P.page_advance(plan, lengths)
        for r, n in enumerate(new):
            outs[r].append(o[sum(new[:r]):sum(new[:r]) + n])
            at[r] += n
    assert lengths.tolist() == [23, 0, 50] and held.tolist() == [2, 0, 4] and n_free.tolist() == [2]
    for r, n in enumerate(total):
        x = qkv[r].cpu().double()

        def turned(y):
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)
            ang = torch.arange(n).double()[:, None, None] * freq.cpu()
            lo, hi = y[..., :rd // 2], y[..., rd // 2:rd]
            return torch.cat([lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin(), y[..., rd:]], -1).to(dtype)
        q, k, v = turned(x[:, :H]), turned(x[:, H:H + G]), qkv[r].cpu()[:, H + G:]
        pages = -(-n // page)
        kk, vv = (torch.zeros(pages * page, G, hd, dtype=dtype) for _ in range(2))
        kk[:n], vv[:n] = k, v
        one = (torch.tensor([0, n]), [0], [n])
        want, size, score = R.attention(q, *(y.view(pages, page, G, hd).transpose(1, 2) for y in (kk, vv)),
                                        torch.arange(pages)[None], *one)
        # q and k may each take the other neighbour of 16 bits, which moves a score by 2^-11 of the sum of its terms' sizes twice
        bound = R.attention_bound(want, size, score, dtype, hd, n) + 2 * 2 * 2.0 ** -11 * score * size
        assert bool(((torch.cat(outs[r]).cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("tokens", [4096, 4097, 9001])
def test_page_plan_of_many_tokens(tokens):
    """Sequences that are not served and rows behind the last among thousands of tokens."""
    case = ([2, 0, 2, 4, 1, 3], [3000, 1, 9, 500, 400, 190], [70, 31, 5, 0, 900], [2, 1, 1, 0, 29], 130, 111, tokens, 32)
    requests, new, lengths, held, table, free, n_free, tokens, page = _plan_state(case, R.gen(case))
    d = _on_gpu(requests, new, lengths, held, table, free, n_free)
    got = _paged().page_plan(*d, tokens=tokens, page_size=page)
    want, n_free = R.plan(requests, new, lengths, held, table, free, n_free, tokens, page)
    assert [x >= 0 for x in want[1]] == [True, True, False, True, False, False]
    for name, x, y in zip(got._fields, got, want):
        assert x.tolist() == y, name
    assert d[4].tolist() == table and d[6].tolist() == [n_free]


def test_caches_past_32_bits():
    """Pages whose first element lies past 2^31 and past 2^32 bytes: as in a small cache."""
    P = _paged()
    H, G, hd, page, N = 8, 8, 256, 256, 300
    g = R.gen("far")
    x = torch.randn(N, H + 2 * G, hd, generator=g).to(BF16).cuda()
    w = torch.ones(hd, dtype=BF16, device="cuda")
    freq = (1e4 ** (-torch.arange(0, hd, 2).double() / hd)).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    n_pages = 2 ** 31 // (G * page * hd) + 3
    outs = []
    for pages in (3, n_pages):
        kp, vp = (torch.empty(pages, G, page, hd, dtype=BF16, device="cuda") for _ in range(2))
        for c in (kp, vp):
            c[-3:].zero_()
        table = torch.tensor([[pages - 1, pages - 3]], **i32)
        pos = torch.arange(N, device="cuda")
        slots = table[0][pos // page].long() * page + pos % page
        plan = P.PagePlan(torch.tensor([0, N], **i32), torch.tensor([0], **i32), torch.tensor([N], **i32), pos, slots)
        q = P.paged_write(x[:, :H], x[:, H:H + G], x[:, H + G:], w, w, freq, kp, vp, pos, slots, eps=1e-6)
        one = P.PagePlan(torch.tensor([0, 1], **i32), *plan[1:3], pos[-1:], slots[-1:])
        outs.append((q, kp[-3:].clone(), vp[-3:].clone(), P.attn_paged(q, kp, vp, table, plan), P.attn_paged(q[-1:], kp, vp, table, one, max_new=1)))
        del kp, vp
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_a_captured_step_of_all_kinds():
    """Plan, write, attend, recur and advance in one graph: every replay as the eager calls, which run between them on
    states of their own."""
    P = _paged()
    H, G, hd, page, N, hk, hv, dk = 6, 2, 64, 16, 100, 2, 4, 64
    g = R.gen("captured")
    conv_dim = 2 * hk * dk + hv * dk
    x, z, ab = (torch.randn(N, n, generator=g).to(F16).cuda() for n in ((H + 2 * G) * hd + conv_dim, hv * dk, 2 * hv))
    qkv = x[:, :(H + 2 * G) * hd].view(N, H + 2 * G, hd)
    w, nw = torch.ones(hd, dtype=F16, device="cuda"), torch.ones(dk, dtype=F16, device="cuda")
    freq = (1e4 ** (-torch.arange(0, 32, 2).double() / 32)).cuda()
    conv_w = (0.5 * torch.randn(conv_dim, 4, generator=g)).to(F16).cuda()
    ssm_a, dt_bias = -torch.ones(hv, device="cuda"), torch.zeros(hv, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    new = torch.zeros(3, **i32)
    requests = torch.tensor([3, 0, 1], **i32)

    def state():
        kp, vp = (torch.zeros(40, G, page, hd, dtype=F16, device="cuda") for _ in range(2))
        return dict(kp=kp, vp=vp, lengths=torch.zeros(4, **i32), held=torch.zeros(4, **i32), table=torch.full((4, 12), -1, **i32),
                    free=torch.arange(40, **i32), n_free=torch.tensor([40], **i32),
                    conv=torch.zeros(4, 3, conv_dim, dtype=F16, device="cuda"), rec=torch.zeros(4, hv, dk, dk, device="cuda"))

    def step(s):
        plan = P.page_plan(requests, new, s["lengths"], s["held"], s["table"], s["free"], s["n_free"], tokens=N, page_size=page)
        q = P.paged_write(qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], w, w, freq, s["kp"], s["vp"], plan.pos, plan.slots, eps=1e-6)
        a = P.attn_paged(q, s["kp"], s["vp"], s["table"], plan)
        o = P.gdn_packed(x[:, -conv_dim:], z, ab, s["conv"], conv_w, ssm_a, dt_bias, s["rec"], nw, plan, key_heads=hk, value_heads=hv,
                         head_k_dim=dk, head_v_dim=dk, eps=1e-6)
        P.page_advance(plan, s["lengths"])
        return [*plan, a, o]
    captured, eager = state(), state()
    step(state())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(captured)
    for i, n in enumerate(([30, 0, 1], [1, 70, 20], [1, 1, 1], [80, 3, 17], [500, 1, 1])):
        new.copy_(torch.tensor(n, **i32))
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        for j, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a.nan_to_num(nan=7.), b.nan_to_num(nan=7.)), (i, j)
        for name in eager:
            assert torch.equal(captured[name], eager[name]), (i, name)
    assert eager["lengths"].tolist() == [74, 39, 0, 112]
