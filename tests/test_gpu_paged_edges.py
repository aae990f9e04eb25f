"""Steps of packed requests over paged caches where they can go wrong: bits of softmax weights and of small rows and
columns, values that are not finite, steps without sequences, and steps of hundreds of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

import paged_ref as R  # noqa: E402
from test_gpu_paged import _attend, _attn_inputs, _check_attn, _check_gdn, _gdn_inputs, _name, _paged, _run_gdn  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


# ---- attention: bits of the weights ----------------------------------------------------------------

@pytest.mark.parametrize("rep", [1, 16, 48], ids=["row", "few", "many"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_weights_keep_22_bits(dtype, hd, rep):
    """V rows whose weighted sum cancels: outputs are the weights' last bits. They keep 22 for both types, as the operators
    over one sequence hold them."""
    L = 6
    q, kp, vp, table, plan, _ = _attn_inputs([L - 1] * 32, [1] * 32, 16, rep, 1, hd, dtype, key=("bits", hd, rep), k_size=0.02)
    q[:] = q[:, :1]  # one row of scores for all heads of a sequence
    for b in range(32):
        page = int(table[plan[1][b], 0])
        k = kp[page, 0, :L].double()
        p = torch.softmax(k @ q[b, 0].double() / hd ** 0.5, 0)
        left = torch.zeros(hd, dtype=torch.float64)
        for j in range(L):  # each takes what those before it leave, but for its rounding
            if j:
                vp[page, 0, j] = (-left / p[j]).to(dtype)
            left += p[j] * vp[page, 0, j].double()
    got = _attend(q, kp, vp, table, plan)
    want, size, score = R.attention(q, kp, vp, table, *plan[:3])
    bound = R.attention_bound(want, size, score, dtype, hd, L)
    if dtype is BF16:
        bound -= (2.0 ** -16 - 2.0 ** -22) * size
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_positions_of_no_weight_add_nothing(dtype):
    """A first position that everybody looks at, 60000 behind it with weights e^-40 of its own and a large V: nothing of
    that V reaches the outputs. 512 single tokens, then a prompt, each enough to leave the positions in long pieces; the
    sequences share their pages."""
    L, hd, P = 60000, 64, _paged()
    kp, vp = torch.full((235, 1, 256, hd), -2.5, dtype=dtype, device="cuda"), torch.full((235, 1, 256, hd), 1000.0, dtype=dtype, device="cuda")
    kp[0, 0, 0], vp[0, 0, 0] = 2.5, 0.0
    i32 = dict(dtype=torch.int32, device="cuda")
    for B, n, heads in ((512, 1, 4), (1, 8192, 64)):
        table = torch.arange(235, **i32).expand(B, -1).contiguous()
        cu, rows, lens = torch.arange(B + 1, **i32) * n, torch.arange(B, **i32), torch.full((B,), L, **i32)
        q = torch.ones(B * n, heads, hd, dtype=dtype, device="cuda")
        # 60000 * 1000 * e^-40 = 3e-10; a V of 1000 at 2^-33 of the first one's weight for each position would be 7e-3
        assert float(P.attn_paged(q, kp, vp, table, P.PagePlan(cu, rows, lens, rows, rows), max_new=n).abs().max()) <= 1e-6


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_small_weights_behind_a_large_one(dtype):
    """A first position that takes nearly all weight and has no V, 60000 behind it with 2^-29.4 of its weight each, which
    make the output. In fp16 a weight's last place is 2^-38 of the largest, as in the attention over one sequence."""
    L, hd, P = 60000, 64, _paged()
    kp, vp = torch.full((235, 1, 256, hd), -0.0435, dtype=dtype, device="cuda"), torch.full((235, 1, 256, hd), 1000.0, dtype=dtype, device="cuda")
    kp[0, 0, 0], vp[0, 0, 0] = 2.5, 0.0
    small = torch.exp((kp[0, 0, 1].double() - 2.5).sum() / 8)
    i32 = dict(dtype=torch.int32, device="cuda")
    for B, n, heads in ((512, 1, 4), (1, 8192, 64)):
        table = torch.arange(235, **i32).expand(B, -1).contiguous()
        cu, rows, lens = torch.arange(B + 1, **i32) * n, torch.arange(B, **i32), torch.full((B,), L, **i32)
        q = torch.ones(B * n, heads, hd, dtype=dtype, device="cuda")
        got = P.attn_paged(q, kp, vp, table, P.PagePlan(cu, rows, lens, rows, rows), max_new=n)[0].double()
        seen = L - n  # by the first token
        want = seen * small * 1000 / (1 + seen * small)
        # half a last place of each, 22 bits, the sums' roundings (2^-23 for 8 terms), one rounding of the output
        bound = 2.0 ** -39 * seen * 1000 + (2.0 ** -22 + (seen / 8 + 100) * 2.0 ** -23 + torch.finfo(dtype).eps / 2) * want
        assert bool(((got - want).abs() <= bound).all()), float((got - want).abs().max() / bound)


# ---- attention: values that are not finite ---------------------------------------------------------

@pytest.mark.parametrize("at", [0, 20, 34, 40], ids=["block before", "middle", "last block", "own"])
@pytest.mark.parametrize("cached", [40, 300])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_single_token_sees_what_is_not_finite(hd, value, cached, at):
    """V of infinity at a position that a single token sees is its output, wherever in its blocks that is."""
    at += cached - 40
    for dtype in (F16, BF16):
        q, kp, vp, table, plan, gate = _attn_inputs([cached, 3], [1, 1], 16, 6, 2, hd, dtype, key=("one", hd, cached), k_size=0.1)
        row = int(plan[1][0])
        vp[table[row, at // 16], :, at % 16, 5] = value
        for g in (None, gate):
            got = _attend(q, kp, vp, table, plan, g)
            keep = torch.arange(hd) != 5
            assert bool(torch.isfinite(got[0][:, keep]).all()) and bool(torch.isfinite(got[1]).all())
            assert bool((torch.isnan(got[0][:, 5]) if value != value else got[0][:, 5] == value).all())


@pytest.mark.parametrize("cached", [0, 700])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_prompts_add_up_what_is_not_finite(dtype, hd, cached):
    """A prompt's rows that see a V of infinity among places that others do not see: NaN where the row is NaN for another
    reason (a score, a gate, an infinity of the other sign), infinite elsewhere; the gate's sign and NaN count."""
    n = 60
    q, kp, vp, table, plan, gate = _attn_inputs([cached], [n], 16, 6, 1, hd, dtype, key=("sum", hd, cached), k_size=0.1)
    row = int(plan[1][0])

    def at(t, p=cached):
        return table[row, (p + t) // 16], 0, (p + t) % 16
    vp[at(30)][5] = INF
    vp[at(40)][5] = -INF
    vp[at(20)][7] = -INF
    q[50, 2, 0] = NAN
    gate[25, 1, hd + 7], gate[33, 0, hd + 5], gate[34, 0, hd + 5] = NAN, NAN, -INF
    if cached:  # seen by all
        vp[at(0, 100)][9] = INF
        vp[at(45)][9] = -INF
    want = torch.zeros(n, 6, hd)
    want[30:, :, 5] = INF
    want[40:, :, 5] = NAN
    want[20:, :, 7] = -INF
    if cached:
        want[:, :, 9] = INF
        want[45:, :, 9] = NAN
    want[50, 2] = NAN
    for g in (None, gate):
        w = want.clone()
        if g is not None:
            w[25, 1, 7] = w[33, 0, 5] = w[34, 0, 5] = NAN
        got = _attend(q, kp, vp, table, plan, g)
        odd = ~torch.isfinite(w)
        assert torch.equal(torch.isfinite(got), ~odd)
        assert torch.equal(got[odd].float().nan_to_num(nan=7.0), w[odd].nan_to_num(nan=7.0))


# ---- steps of many sequences, and of none ----------------------------------------------------------

@pytest.mark.parametrize("N", [1, 16, 100])
def test_steps_without_sequences(N):
    """No sequence at all: every row lies behind the last."""
    P = _paged()
    i32, i64 = torch.int32, torch.int64
    none = P.PagePlan(torch.zeros(1, dtype=i32).cuda(), torch.zeros(0, dtype=i32).cuda(), torch.zeros(0, dtype=i32).cuda(),
                      torch.full((N,), -1, dtype=i64).cuda(), torch.full((N,), -1, dtype=i64).cuda())
    for hint in ({}, {"max_new": 1}):
        pages = torch.ones(3, 2, 16, 64, dtype=F16, device="cuda")
        got = P.attn_paged(torch.ones(N, 4, 64, dtype=F16, device="cuda"), pages, pages, torch.zeros(2, 4, dtype=i32, device="cuda"), none, **hint)
        assert got.shape == (N, 4, 64) and not bool(got.any())
        case = ([], [], 2, 4, 64, 64, 4, F16)
        t, _ = _gdn_inputs(case)
        t = tuple(torch.ones(N, x.shape[1], dtype=F16) for x in t[:3]) + t[3:]
        out, conv, rec = _run_gdn(case, t, none, **hint)
        assert out.shape == (N, 256) and not bool(out.any()) and torch.equal(conv, t[3]) and torch.equal(rec, t[7])


def _crowd(B, longest, seed):
    """(cached, new, sequences that are not served) of a step of B sequences: single tokens, some without any, some of a few,
    some prompts; one that is not served among each 64; long ones on both sides of each border of 64."""
    g = R.gen("crowd", B, seed)
    cached = torch.randint(0, 200, (B,), generator=g).tolist()
    new = [1] * B
    for b in torch.randperm(B, generator=g)[:B // 4].tolist():
        new[b] = int(torch.randint(0, 30, (1,), generator=g))
    for b in range(0, B, 64):
        for at, c, n in ((b - 2, longest, 1), (b + 1, longest // 2, 1), (b + 3, longest, 45), (b + 5, 0, 70)):
            if 0 <= at < B:
                cached[at], new[at] = c, n
    return cached, new, [b for b in (7, 71, 135, 199, 263, 1000) if b < B]


# (sequences, longest context, page, heads, kv heads, head dim, dtype)
CROWDS = [(64, 3000, 16, 4, 2, 64, F16), (65, 3000, 16, 4, 2, 64, BF16), (130, 5000, 64, 6, 1, 128, F16), (300, 2000, 32, 4, 1, 256, BF16),
          (1024, 700, 16, 2, 1, 64, F16)]


@pytest.mark.parametrize("case", CROWDS, ids=_name)
def test_attention_of_many_sequences(case):
    B, longest, page, H, G, hd, dtype = case
    cached, new, gone = _crowd(B, longest, 0)
    q, kp, vp, table, plan, gate = _attn_inputs(cached, new, page, H, G, hd, dtype, key=case, tail=2)
    plan = [x.clone() for x in plan]
    plan[1][gone] = -1
    cu, N = plan[0].tolist(), q.shape[0] - 2
    lost = torch.zeros(N, dtype=torch.bool)
    for b in gone:
        lost[cu[b]:cu[b + 1]] = True
    want, size, score = R.attention(q[:N], kp, vp, table, *plan[:3], gate[:N, :, hd:])
    bound = R.attention_bound(want, size, score, dtype, hd, longest + 70)
    for hint in ({}, {"max_new": 1}):  # in both kinds of workgroups, and in one
        got = _attend(q, kp, vp, table, plan, gate, **hint)
        assert not bool(got[N:].any()) and bool(torch.isnan(got[:N][lost]).all())
        err = (got[:N].double() - want).abs()
        assert bool((err <= bound)[~lost].all()), float((err - bound)[~lost].max())


def test_a_prompt_is_cut_alike_beside_any_number_of_single_tokens():
    """How a chunk of a prompt behind many positions is cut into pieces follows from the sequences of many rows: its bits are
    the same beside 3 single tokens and beside 100."""
    P, H, G, hd, page, long, n = _paged(), 6, 1, 128, 64, 20000, 50
    g = R.gen("alike")
    pages = -(-(long + n) // page)
    kp, vp = (torch.randn(pages, G, page, hd, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(n + 1100, H, hd, generator=g).half().cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    got = []
    for singles, at in ((3, 0), (62, 30), (63, 63), (64, 64), (100, 5), (1023, 1000)):  # the chunk behind `at` of them
        new = [1] * at + [n] + [1] * (singles - at)
        cu = torch.tensor([0] + new).cumsum(0).int().cuda()
        lens = torch.tensor([200] * at + [long + n] + [200] * (singles - at), **i32)
        table = torch.arange(pages, **i32).expand(singles + 1, -1).contiguous()
        plan = P.PagePlan(cu, torch.arange(singles + 1, **i32), lens, None, None)
        x = torch.cat([q[n:n + at], q[:n], q[n + at:n + singles]])
        got.append(P.attn_paged(x, kp, vp, table, plan)[at:at + n])
    for x in got[1:]:
        assert torch.equal(x, got[0])


@pytest.mark.parametrize("turns", [16, 17, 70])
def test_attention_of_many_turns(turns):
    """Turns of some tokens behind long contexts, more than the search for pieces takes, between single tokens."""
    new, cached = [1, 9] * turns, [40, 0] * turns
    cached[1::2] = [1500 + 61 * i % 900 for i in range(turns)]
    q, kp, vp, table, plan, gate = _attn_inputs(cached, new, 32, 4, 1, 64, F16, key=("turns", turns))
    _check_attn(_attend(q, kp, vp, table, plan, gate), q, kp, vp, table, plan, gate)


@pytest.mark.parametrize("B", [64, 65, 130, 300, 1024])
def test_recurrence_of_many_sequences(B):
    cached, new, gone = _crowd(B, 500, 1)
    case = (cached, new, 1, 2, 32, 64, 4, F16 if B % 2 else BF16)
    t, plan = _gdn_inputs(case, tail=2)
    plan = [x.clone() for x in plan]
    rows = plan[1].clone()
    plan[1][gone] = -1
    cu, N = plan[0].tolist(), t[0].shape[0] - 2
    lost = torch.zeros(N, dtype=torch.bool)
    for b in gone:
        lost[cu[b]:cu[b + 1]] = True
    cut = tuple(x[:-2] for x in t[:3]) + t[3:]
    for hint in ({}, {"max_new": 1}):  # long ones by chunks, and all token by token
        out, conv, rec = _run_gdn(case, t, plan, **hint)
        assert not bool(out[N:].any()) and bool(torch.isnan(out[:N][lost]).all())
        kept = [int(rows[b]) for b in gone]
        assert torch.equal(conv[kept], t[3][kept]) and torch.equal(rec[kept], t[7][kept])
        _check_gdn(case, cut, plan, (out[:N].masked_fill(lost[:, None], 0), conv, rec))


# ---- GatedDeltaNet: small rows and columns ---------------------------------------------------------

def _one_head(n, K=4, dv=64, dk=128):
    """One head of n tokens from a cached state, its convolution the current token's input alone, so that its outputs have
    their inputs' bits. Returns the call's tensors (test_gpu_paged._gdn_inputs) and the plan."""
    case = ([5], [n], 1, 1, dk, dv, K, BF16)
    t, plan = _gdn_inputs(case)
    t = [x.clone() for x in t]
    t[4].zero_()
    t[4][:, -1] = 1
    t[5][:], t[6][:] = -0.05, 0.0
    return case, t, plan


@pytest.mark.parametrize("size", [1e-5, 1e-7, 1e-9, 1e-15])
@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("n", [1, 9, 16, 130])
def test_small_rows_keep_their_bits(n, which, size):
    """q or k rows far below the norm's epsilon enter the recurrence with float32's bits: with small q the outputs, with
    small k what the state gains from zero, relative to what they are."""
    case, t, plan = _one_head(n)
    dk, dv = 128, 64
    cols = slice(0, dk) if which == "q" else slice(dk, 2 * dk)
    t[0][:, cols] = (t[0][:, cols].float() * size).bfloat16()
    if which == "k":
        plan = list(plan)
        plan[2] = torch.tensor([n], dtype=torch.int32)  # from zeros
    out, conv, rec = _run_gdn(case, t, plan)
    want, _, want_rec, scale = R.gdn(*t, *plan[:3], 1, 1, dk, dv, 1e-6)
    r = int(plan[1][0])
    # float32: 16 roundings on the way to q and k, sums of 128 rows and of up to n tokens. Matrix cores truncate:
    # 2^-22 for every 8 terms
    rel = (16 + dk / 8 + n / 4) * 2.0 ** -22
    if which == "k":
        # rows of the state are sums of k_t u_t, u_t at most 2 |v_t| (k is small: what the state gives back is smaller still)
        x = t[0].double()
        k = x[:, cols]
        k = (k * torch.sigmoid(k)).abs()
        k = k / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt() / dk ** 0.5
        v = x[:, 2 * dk:]
        terms = k.T @ (2 * (v * torch.sigmoid(v)).abs())
        err = (rec[r, 0].double() - want_rec[r, 0]).abs()
        assert bool((err <= rel * terms).all()), float((err / terms).max())
        assert float(want_rec[r].abs().max()) > 0
    else:
        # an output is a sum over rows of q_i S_i: sizes from the largest entry of the state on its way
        x = t[0].double()[:, cols]
        q = (x * torch.sigmoid(x)).abs()
        q = q / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt() / dk
        top = float(t[7][r].abs().max()) + 2 * float(t[0][:, 2 * dk:].abs().max()) * n ** 0.5
        # o over the norm's root, which is at least 1e-3
        terms = q.sum(-1, keepdim=True) * top * 1e3 * scale
        err = (out.double() - want).abs()
        assert bool((err <= torch.finfo(BF16).eps / 2 * want.abs() + rel * terms).all()), float(((err - 2.0 ** -8 * want.abs()) / terms).max())


@pytest.mark.parametrize("n", [2, 16, 64, 200])
def test_columns_of_a_state_do_not_meet(n):
    """Columns of the state, and of v, from 1 down to 1e-7 of their neighbours: each keeps the bits of its own size."""
    case, t, plan = _one_head(n)
    dk, dv = 128, 64
    size = 10.0 ** -(torch.arange(dv) % 8).float()
    size = size[torch.randperm(dv, generator=R.gen("columns"))]
    t[0][:, 2 * dk:] = (t[0][:, 2 * dk:].float() * size).bfloat16()
    t[7] = t[7] * size
    out, conv, rec = _run_gdn(case, t, plan)
    want, _, want_rec, scale = R.gdn(*t, *plan[:3], 1, 1, dk, dv, 1e-6)
    r = int(plan[1][0])
    # as test_gpu_paged._check_gdn's bound, each column by itself: its largest entry, of v too
    top = torch.maximum(want_rec[r, 0].abs().amax(0), t[7][r, 0].double().abs().amax(0)) + 2 * t[0][:, 2 * dk:].double().abs().amax(0)
    err = (rec[r, 0].double() - want_rec[r, 0]).abs()
    assert bool((err <= (n + 16) * 2.0 ** -21 * top).all()), float((err / top).max())
