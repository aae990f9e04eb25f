"""The 8-bit K/V cache (``kv8_write``, ``kv8_read``, ``attn_kv8``) against its definition in float64:
rows around the 16-row tiles and positions around the 32-position blocks, ragged batches, trees of
drafted tokens, positions split over workgroups, values that are not finite, and rows outside the cache."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

F16, BF16 = torch.float16, torch.bfloat16


def _gen(*key):
    return torch.Generator().manual_seed(hash(key) % (1 << 31))


def _quantise(x):
    """(bytes, float32 scales) of rows x (float64), by the definition."""
    scale = (x.abs().amax(-1) / 127).float()
    u = (x / scale.double()[..., None]).round().clamp(-127, 127) + 128
    u = torch.where(scale[..., None] > 0, u, 128.0)
    bad = ~torch.isfinite(x).all(-1)
    u[bad] = 128.0
    return u.to(torch.uint8), torch.where(bad, float("nan"), scale)


def _values(u, scale):
    return (u.double() - 128) * scale.double()[..., None]


def _chain(parents, t):
    """Node t and its ancestors."""
    out = [t]
    while parents[out[-1]] >= 0:
        out.append(int(parents[out[-1]]))
    return out


def _tree(B, S, gen, kind="random"):
    t = torch.arange(S).expand(B, S)
    if kind == "chain":
        p = t - 1
    elif kind == "star":
        p = torch.full((B, S), -1)
    else:
        p = (t - 1 - (torch.rand(B, S, generator=gen) * 5).long()).clamp(min=-1)
    return p.to(torch.int32)


# ---- writing and reading back --------------------------------------------------------------------

# (batch, tokens, positions, cache length, heads, kv heads, head dim, rotary dim, dtype, tree)
WRITES = [(1, 1, [0], 1, 1, 1, 64, 0, F16, None), (1, 1, [5], 9, 24, 4, 256, 64, F16, None),
          (3, 7, [0, 9, 4], 16, 6, 2, 128, 128, BF16, None), (2, 33, [40], 80, 4, 4, 64, 6, F16, None),
          (1, 300, [70001], 70400, 12, 2, 256, 64, BF16, None), (2, 64, [3, 100], 200, 5, 1, 128, 32, F16, "random"),
          (1, 17, [1000], 1017, 8, 8, 256, 256, BF16, "star"), (4, 512, [0], 512, 2, 1, 64, 16, BF16, None)]


def _write_inputs(case):
    B, S, pos, L, H, G, hd, rd, dtype, tree = case
    g = _gen(B, S, hd)

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(dtype)
    rows = rnd(B, S, H * 2 * hd + 2 * G * hd + 2)  # q | k | v of one product, and a row stride that is not a power of two
    n = H * 2 * hd
    freq = 1e7 ** (-torch.arange(0, rd, 2).double() / max(rd, 1))
    u = torch.randint(0, 256, (2, B, G, L, hd), generator=g, dtype=torch.uint8)
    sc = torch.rand(2, B, G, L, generator=g)
    return (rows[..., :n], rows[..., n:n + G * hd], rows[..., n + G * hd:n + 2 * G * hd], (2 + rnd(hd)), (2 + rnd(hd)), freq,
            u[0], u[1], sc[0], sc[1], torch.tensor(pos), None if tree is None else _tree(B, S, g, tree))


def _norm_rope(x, w, at, freq, rd, eps):
    """float64 rows x (B, S, n, hd) at positions at (B, S)."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    ang = at.double()[..., None, None] * freq
    lo, hi = x[..., :rd // 2], x[..., rd // 2:rd]
    return torch.cat([lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin(), x[..., rd:]], -1)


def _run_write(case, t, **kw):
    from mlx_gsq_amd.runtime.kernels import kv8
    B, S, pos, L, H, G, hd, rd, dtype, tree = case
    rows = torch.cat([t[0], t[1], t[2], t[0][..., :2]], -1).cuda()
    n = H * 2 * hd
    d = [x.cuda().clone() for x in t[3:11]]
    q = kv8.kv8_write(rows[..., :n], rows[..., n:n + G * hd], rows[..., n + G * hd:n + 2 * G * hd], *d, heads=H,
                      kv_heads=G, head_dim=hd, rotary_dim=rd, eps=1e-6, parents=None if t[11] is None else t[11].cuda(), **kw)
    return q.cpu(), [x.cpu() for x in d[3:7]]


@pytest.mark.parametrize("case", WRITES, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
def test_kv8_write_matches_definition(case):
    B, S, pos, L, H, G, hd, rd, dtype, tree = case
    t = _write_inputs(case)
    q, (kc, vc, ks, vs) = _run_write(case, t)
    p = torch.tensor(pos).expand(B)
    if tree is None:
        depth = torch.arange(S).expand(B, S)
    else:
        depth = torch.tensor([[len(_chain(t[11][b], i)) - 1 for i in range(S)] for b in range(B)])
    at = p[:, None] + depth
    want_q = _norm_rope(t[0].double().reshape(B, S, H, 2 * hd)[..., :hd], t[3], at, t[5], rd, 1e-6)
    k = _norm_rope(t[1].double().reshape(B, S, G, hd), t[4], at, t[5], rd, 1e-6)
    ku, kscale = _quantise(k)
    vu, vscale = _quantise(t[2].double().reshape(B, S, G, hd))
    # q: one rounding to dtype, after a norm and a rotation in float32: 16 roundings of the row's size
    err = (q.double().view(B, S, H, hd) - want_q).abs()
    eps = torch.finfo(dtype).eps / 2
    assert bool((err <= eps * want_q.abs() + 16 * 2.0 ** -24 * want_q.abs().amax(-1, keepdim=True) + 2.0 ** -25).all())
    want = [t[6].clone(), t[7].clone(), t[8].clone(), t[9].clone()]
    for b in range(B):
        rows = slice(int(p[b]), int(p[b]) + S)
        for c, new in zip(want, (ku, vu, kscale, vscale)):
            c[b, :, rows] = new[b].transpose(0, 1)
    # k is formed in float64 on both sides: bytes differ where x / s is within rounding of a border only
    border = torch.zeros_like(kc, dtype=torch.bool)
    for b in range(B):
        x = (k / kscale.double()[..., None])[b].transpose(0, 1)
        border[b, :, int(p[b]):int(p[b]) + S] = ((x - x.floor()) - 0.5).abs() < 1e-9
    assert torch.equal(kc[~border], want[0][~border]) and int(border.sum()) < 1 + 1e-6 * kc.numel()
    # the scale of K: a float32 rounding of values that agree to 1e-15
    assert torch.equal(vc, want[1]) and torch.equal(vs, want[3])
    assert bool(((ks - want[2]).abs() <= 2.0 ** -23 * want[2].abs()).all()) and float((ks != want[2]).double().mean()) < 1e-3


def test_kv8_write_not_finite_and_zero_rows():
    """Rows that hold a NaN or an infinity stand for NaN, zero rows for zeros; other rows do not change."""
    case = (1, 9, [3], 20, 2, 2, 64, 16, F16, None)
    t = list(_write_inputs(case))
    t[2] = t[2].clone()
    clean_q, clean = _run_write(case, t)
    t[1] = t[1].clone()
    t[1][0, 2, 5] = float("nan")            # k of token 2, head 0
    t[2][0, 4, 64 + 7] = float("inf")       # v of token 4, head 1
    t[2][0, 6, :64] = 0.0                   # v of token 6, head 0
    q, (kc, vc, ks, vs) = _run_write(case, t)
    assert torch.equal(q, clean_q)
    assert torch.isnan(ks[0, 0, 5]) and bool((kc[0, 0, 5] == 128).all())
    assert torch.isnan(vs[0, 1, 7]) and bool((vc[0, 1, 7] == 128).all())
    assert float(vs[0, 0, 9]) == 0.0 and bool((vc[0, 0, 9] == 128).all())
    keep = torch.ones(1, 2, 20, dtype=torch.bool)
    keep[0, 0, 5] = False
    assert torch.equal(kc[keep], clean[0][keep]) and torch.equal(ks[keep], clean[2][keep])
    keep[0, 0, 5], keep[0, 1, 7], keep[0, 0, 9] = True, False, False
    assert torch.equal(vc[keep], clean[1][keep]) and torch.equal(vs[keep], clean[3][keep])


def test_kv8_write_ties_and_tiny_scales():
    """v rows whose quotients fall on a half (rounded to even), and rows so small that the scale is
    subnormal or rounds to zero (bytes clamped to 1 .. 255)."""
    hd = 64
    case = (1, 4, [0], 4, 1, 1, hd, 0, BF16, None)
    t = list(_write_inputs(case))
    v = torch.zeros(1, 4, hd)
    v[0, 0] = (torch.arange(hd) - 32) + 0.5  # with a largest value of 127: x / s = x
    v[0, 0, 0] = 127.0
    v[0, 1] = 3 * v[0, 0]
    v[0, 2, :3] = torch.tensor([1.5, -1.0, 0.25]) * 2.0 ** -125
    v[0, 3, 0] = 2.0 ** -133                 # largest / 127 is under half of the smallest float32
    t[2] = v.to(BF16)
    _, (kc, vc, ks, vs) = _run_write(case, t)
    u, s = _quantise(t[2].double().view(1, 4, 1, hd))
    assert torch.equal(vc[0, 0], u[0, :, 0]) and torch.equal(vs[0, 0], s[0, :, 0])


def test_kv8_read():
    from mlx_gsq_amd.runtime.kernels import kv8
    for B, G, L, hd, start, n in ((1, 1, 1, 64, 0, 1), (2, 3, 37, 128, 5, 20), (1, 4, 1000, 256, 999, 1), (2, 2, 65, 64, 0, 65),
                                  (1, 1, 8, 64, 3, 0)):
        g = _gen(B, L, hd)
        u = torch.randint(0, 256, (2, B, G, L, hd), generator=g, dtype=torch.uint8)
        s = torch.rand(2, B, G, L, generator=g) * 0.1
        s[0, 0, 0, L - 1] = float("nan")
        d, ds = u.cuda(), s.cuda()
        for dtype in (torch.float32, F16, BF16):
            k, v = kv8.kv8_read(d[0], d[1], ds[0], ds[1], dtype=dtype, start=start, length=n)
            for got, uu, ss in ((k, u[0], s[0]), (v, u[1], s[1])):
                want = ((uu.float() - 128) * ss[..., None])[:, :, start:start + n].to(dtype)
                assert got.shape == want.shape
                assert torch.equal(torch.nan_to_num(got.cpu().float(), 7.0), torch.nan_to_num(want.float(), 7.0))


# ---- attention -----------------------------------------------------------------------------------

def _attn_inputs(B, S, pos, L, H, G, hd, dtype, tree=None):
    g = _gen(B, S, L, hd, H)

    def rnd(*shape):
        return torch.randn(*shape, generator=g)
    k, ks = _quantise(rnd(B, G, L, hd).double())
    v, vs = _quantise((rnd(B, G, L, hd) * torch.exp(rnd(B, G, L, 1))).double())
    return {"q": rnd(B, S, H * hd).to(dtype), "qg": rnd(B, S, H * 2 * hd).to(dtype), "k": k, "v": v, "ks": ks, "vs": vs,
            "pos": torch.tensor(pos), "parents": None if tree is None else _tree(B, S, g, tree)}


def _attn(t, H, G, hd, long=False, **kw):
    """``long``: in caches long enough that the tile kernel is chosen (49152 tiles of 16 rows x blocks of 32
    positions, for more than 32 rows of a KV head), which hold anything behind the tokens."""
    from mlx_gsq_amd.runtime.kernels import kv8
    d = {n: None if x is None else x.cuda() for n, x in t.items()}
    if long:
        B, S = t["q"].shape[:2]
        tiles = -(-S * (H // G) // 16) * B * G
        assert S * (H // G) > 32
        for n in ("k", "v", "ks", "vs"):
            x = d[n]
            d[n] = x.new_full((B, G, max(x.shape[2], 32 * -(-49152 // tiles) + S), *x.shape[3:]), 255 if x.dtype == torch.uint8 else
                              float("inf" if n == "vs" else "nan"))
            d[n][:, :, :x.shape[2]] = x
    return kv8.attn_kv8(d["q"], d["qg"], d["k"], d["v"], d["ks"], d["vs"], d["pos"], heads=H, kv_heads=G, head_dim=hd,
                        parents=d["parents"], **kw).cpu()


def _reference(t, H, G, hd):
    """(out, bound of the error before the last rounding) in float64."""
    B, S = t["q"].shape[:2]
    q, gate = t["q"].double().view(B, S, H, hd), torch.sigmoid(t["qg"].double().view(B, S, H, 2 * hd)[..., hd:])
    out, tol = torch.empty(B, S, H, hd, dtype=torch.float64), torch.empty(B, S, H, hd, dtype=torch.float64)
    bf = t["q"].dtype == BF16
    for b in range(B):
        p0 = int(t["pos"].expand(B)[b])
        n = p0 + S
        see = torch.arange(n)[None, :] <= p0 + torch.arange(S)[:, None]
        if t["parents"] is not None:
            see[:, p0:] = False
            for i in range(S):
                see[i, [p0 + a for a in _chain(t["parents"][b], i)]] = True
        for h in range(H):
            g = h // (H // G)
            k, v = _values(t["k"][b, g, :n], t["ks"][b, g, :n]), _values(t["v"][b, g, :n], t["vs"][b, g, :n])
            sc = torch.matmul(q[b, :, h], k.t().contiguous()) * hd ** -0.5
            p = torch.softmax(sc.masked_fill(~see, float("-inf")), -1)
            out[b, :, h] = torch.matmul(p, v)
            # float32 sums run over bytes u = x / s + 128, not over x, and 128 times the factors' sum is taken off: a term
            # is up to 255 s |factor| in size whatever x is
            ks, vs = (255 * t[x][b, g, :n].double() for x in ("ks", "vs"))
            size = (q[b, :, h].abs().sum(-1, keepdim=True) * ks * see).amax(-1, keepdim=True) * hd ** -0.5
            # a score: float32 sums of hd products in steps of 32 and a few more roundings, absolute; a weight: that in the
            # exponent (over and under the line), exp's and the scales' roundings, one fp16 rounding for bf16
            # outputs; sums over the positions
            weight = 2 * (hd / 32 + 8) * 2.0 ** -24 * size + 8 * 2.0 ** -24 + (2.0 ** -11 if bf else 2.0 ** -21)
            tol[b, :, h] = (weight * torch.matmul(p, v.abs())
                            + (n / 32 + 16) * 2.0 ** -24 * torch.matmul(p, vs)[:, None])
    return out * gate, tol * gate


def _check(got, want, tol, dtype):
    got = got.double().view(want.shape)
    eps = torch.finfo(dtype).eps / 2
    assert torch.isfinite(got).all()
    over = (got - want).abs() - (tol * (1 + eps) + eps * want.abs() + 2.0 ** -25)
    assert float(over.max()) <= 0, float(over.max())


# (batch, tokens, positions, cache length, heads, kv heads, head dim, dtype, tree)
ATTN = [(1, 1, [0], 1, 1, 1, 64, F16, None), (1, 1, [0], 40, 24, 4, 256, F16, None), (1, 1, [31], 64, 6, 1, 256, BF16, None),
        (1, 1, [32], 33, 16, 2, 128, F16, None), (3, 1, [700, 1, 64], 900, 24, 4, 256, F16, None),
        (2, 1, [200], 300, 4, 4, 64, BF16, None), (2, 2, [127, 30], 129, 16, 2, 64, F16, None),
        (1, 5, [10], 20, 40, 8, 128, BF16, None), (1, 3, [333], 400, 24, 4, 256, F16, None),
        (1, 6, [60], 66, 6, 1, 256, BF16, None), (1, 33, [0], 33, 2, 2, 64, F16, None), (2, 70, [0, 13], 90, 12, 2, 256, F16, None),
        (1, 130, [261], 391, 6, 1, 128, BF16, None), (1, 257, [0], 300, 24, 4, 256, F16, None),
        (1, 100, [5], 105, 7, 1, 256, BF16, None),
        (1, 1, [9], 12, 6, 1, 256, F16, "random"), (1, 13, [200], 220, 24, 4, 256, F16, "random"),
        (2, 64, [0, 77], 150, 12, 2, 256, BF16, "random"), (1, 64, [31], 95, 16, 2, 128, F16, "chain"),
        (2, 40, [64], 104, 8, 8, 64, BF16, "star"), (3, 21, [5, 40, 33], 61, 4, 1, 64, F16, "random"),
        (1, 2, [0], 2, 24, 4, 256, F16, "star"), (1, 33, [100], 133, 1, 1, 256, F16, "random")]


def _name(c):
    return "-".join(map(str, c)).replace("torch.", "")


@pytest.mark.parametrize("case", ATTN, ids=_name)
def test_attn_kv8_matches_float64(case):
    B, S, pos, L, H, G, hd, dtype, tree = case
    t = _attn_inputs(B, S, pos, L, H, G, hd, dtype, tree)
    want, tol = _reference(t, H, G, hd)
    # positions behind the new tokens hold anything
    for b in range(B):
        end = int(t["pos"].expand(B)[b]) + S
        t["ks"][b, :, end:], t["vs"][b, :, end:] = float("nan"), float("inf")
    _check(_attn(t, H, G, hd, splits=1), want, tol, dtype)
    _check(_attn(t, H, G, hd), want, tol, dtype)
    if S * (H // G) > 32:
        _check(_attn(t, H, G, hd, long=True, splits=1), want, tol, dtype)


# rows around the 32-row waves and 128-row tiles, positions around the 64-position tiles
TILES = [(1, 33, [0], 33, 1, 1, 256, F16, None), (1, 64, [63], 127, 2, 1, 256, BF16, None), (2, 43, [64, 0], 107, 6, 2, 128, F16, None),
         (1, 129, [1], 130, 1, 1, 64, BF16, None), (3, 21, [95, 200, 31], 221, 24, 4, 256, F16, "random"),
         (1, 64, [0], 64, 16, 2, 128, BF16, "random"), (1, 9, [129], 138, 64, 4, 64, F16, "chain"),
         (1, 300, [700], 1000, 6, 1, 256, F16, None), (2, 100, [0], 100, 40, 8, 256, BF16, None)]


@pytest.mark.parametrize("splits", [1, 2, 5, 64])
@pytest.mark.parametrize("case", TILES, ids=_name)
def test_attn_kv8_tiles(case, splits):
    """The kernel of many rows, whose splits are whole tiles of 64 positions."""
    B, S, pos, L, H, G, hd, dtype, tree = case
    t = _attn_inputs(B, S, pos, L, H, G, hd, dtype, tree)
    want, tol = _reference(t, H, G, hd)
    _check(_attn(t, H, G, hd, long=True, splits=splits), want, tol, dtype)


@pytest.mark.parametrize("tree", [None, "random"])
def test_attn_kv8_tiles_of_256_rows(tree):
    """Head dim 64 with 512 workgroups of them."""
    B, S, pos, L, H, G, hd = 32, 40, [650 - 20 * i for i in range(32)], 700, 16, 16, 64
    t = _attn_inputs(B, S, pos, L, H, G, hd, F16, tree)
    got = _attn(t, H, G, hd, long=True, splits=1)
    for b in (0, 13, 31):
        one = {n: None if x is None else x[b:b + 1] for n, x in t.items()}
        want, tol = _reference(one, H, G, hd)
        _check(got[b:b + 1], want, tol, F16)


@pytest.mark.parametrize("splits", [2, 3, 7, 64])
@pytest.mark.parametrize("case", [(1, 1, [300], 400, 24, 4, 256, F16, None), (2, 1, [0, 900], 1000, 6, 1, 128, BF16, None),
                                  (1, 9, [500], 600, 12, 2, 256, F16, "random"), (2, 50, [90, 3], 200, 6, 2, 64, F16, "random"),
                                  (1, 90, [60], 160, 6, 1, 256, BF16, None)], ids=_name)
def test_attn_kv8_split(case, splits):
    """Positions split over workgroups, some of them without any."""
    B, S, pos, L, H, G, hd, dtype, tree = case
    t = _attn_inputs(B, S, pos, L, H, G, hd, dtype, tree)
    want, tol = _reference(t, H, G, hd)
    _check(_attn(t, H, G, hd, splits=splits), want, tol, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("order", ["rising", "falling", "spread"])
def test_attn_kv8_scores_and_scales_that_move(order, dtype):
    """Scores that rise or fall by 80 over the positions, and V scales over 12 powers of ten with them:
    the references of the exponent and of the scales move in almost every block."""
    B, S, pos, L, H, G, hd = 1, 3, [500], 503, 6, 1, 128
    t = _attn_inputs(B, S, pos, L, H, G, hd, dtype)
    j = torch.arange(L).double() / L
    lvl = {"rising": j, "falling": 1 - j, "spread": (torch.arange(L) % 37).double() / 37}[order]
    t["q"] = torch.full_like(t["q"], 1.0)
    k = torch.ones(B, G, L, hd).double() * (80 / hd ** 0.5) * lvl[:, None]
    t["k"], t["ks"] = _quantise(k)
    v = _values(t["v"], t["vs"]) * (10.0 ** (12 * lvl - 6))[:, None] / 100
    if dtype == F16:
        v = v / 10.0 ** 4
    t["v"], t["vs"] = _quantise(v)
    want, tol = _reference(t, H, G, hd)
    for splits in (1, 4):
        _check(_attn(t, H, G, hd, splits=splits), want, tol, dtype)
    many = dict(t, q=t["q"].repeat(1, 4, 1)[:, :9], qg=t["qg"].repeat(1, 4, 1)[:, :9], pos=torch.tensor([494]))
    want, tol = _reference(many, H, G, hd)
    _check(_attn(many, H, G, hd, long=True, splits=1), want, tol, dtype)


@pytest.mark.parametrize("dtype,power", [(F16, 14), (BF16, 14), (BF16, 45)])
@pytest.mark.parametrize("tree", [None, "random"])
@pytest.mark.parametrize("splits", [1, 3])
def test_attn_kv8_large_values_elsewhere(dtype, power, tree, splits):
    """V rows 2^power times the others', which most rows do not see (later tokens, other branches) or see with a
    probability of next to nothing (keys against the queries): the others are what they would be."""
    B, S, pos, L, H, G, hd = 2, 40, [300, 60], 340, 4, 2, 64
    t = _attn_inputs(B, S, pos, L, H, G, hd, dtype, tree)
    q = t["q"].view(B, S, H, hd)
    q[..., 0] = 32.0
    k, v = _values(t["k"], t["ks"]), _values(t["v"], t["vs"])
    if dtype == F16:
        v = v / 16
    for b in range(B):
        k[b, :, 20:24, 0] = -50.0     # 32 x 50 / 8 = 200 below the others: e^-200
        v[b, :, 20:24] *= 2.0 ** power
        v[b, :, pos[b] + 7::5] *= 2.0 ** power
    t["k"], t["ks"] = _quantise(k)
    t["v"], t["vs"] = _quantise(v)
    want, tol = _reference(t, H, G, hd)
    _check(_attn(t, H, G, hd, splits=splits), want, tol, dtype)
    _check(_attn(t, H, G, hd, long=True, splits=splits), want, tol, dtype)


@pytest.mark.parametrize("power", [-110, -60, 60, 100])
def test_attn_kv8_small_and_large_values(power):
    """bf16 V rows of any size, zeros among them."""
    B, S, pos, L, H, G, hd = 1, 24, [150], 174, 4, 2, 64
    t = _attn_inputs(B, S, pos, L, H, G, hd, BF16)
    t["vs"][:, :, :70] = 0.0
    want, tol = _reference(t, H, G, hd)
    t["vs"] *= 2.0 ** power
    for long in (False, True):
        got = _attn(t, H, G, hd, long=long, splits=1)
        _check((got.double() * 2.0 ** -power), want, tol, BF16)


def test_attn_kv8_bf16_query_sizes():
    """bf16 queries of any size: rows of 2^-60, of 2^40 (with keys to match), and zeros, side by side."""
    B, S, pos, L, H, G, hd = 1, 4, [77], 90, 3, 1, 64
    t = _attn_inputs(B, S, pos, L, H, G, hd, BF16)
    q = t["q"].view(B, S, H, hd).float()
    q[:, 0] *= 2.0 ** -60
    q[:, 1] *= 0.0
    q[:, 2] *= 2.0 ** 40
    t["q"] = q.to(BF16).view(B, S, H * hd)
    t["ks"] = t["ks"] * 2.0 ** -40
    want, tol = _reference(t, H, G, hd)
    _check(_attn(t, H, G, hd, splits=1), want, tol, BF16)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("tree", [None, "random"])
def test_attn_kv8_not_finite(tree, splits, long):
    """A NaN row of the cache, or a query or gate that is not finite, reaches the outputs that see it; every other
    is what it is without it, within the rounding bound (the rows of a wave share when their references
    move, so not bit for bit)."""
    B, S, pos, L, H, G, hd = 2, 40, [50, 61], 110, 4, 2, 64
    t = _attn_inputs(B, S, pos, L, H, G, hd, F16, tree)
    clean, tol = _reference(t, H, G, hd)
    _check(_attn(t, H, G, hd, long=long, splits=splits), clean, tol, F16)

    def sees(b, node):
        if tree is None:
            return [i >= node for i in range(S)]
        return [node in _chain(t["parents"][b], i) for i in range(S)]

    def check(changed, bad):
        got = _attn(dict(t, **changed), H, G, hd, long=long, splits=splits).view(B, S, H, hd)
        assert torch.isnan(got[bad]).all()
        _check(got[~bad], clean[~bad], tol[~bad], F16)
    for name in ("ks", "vs"):
        for node in (7, 33):
            x = t[name].clone()
            x[1, 1, 61 + node] = float("nan")  # a new token of row 1, KV head 1: query heads 2 and 3
            bad = torch.zeros(B, S, H, hd, dtype=torch.bool)
            bad[1, sees(1, node), 2:] = True
            check({name: x}, bad)
        x = t[name].clone()
        x[0, 0, 20] = float("nan")             # a cached token of row 0, KV head 0
        bad = torch.zeros(B, S, H, hd, dtype=torch.bool)
        bad[0, :, :2] = True
        check({name: x}, bad)
    for value in (float("nan"), float("inf")):
        x = t["q"].clone()
        x[0, 12, 3 * hd + 9] = value
        bad = torch.zeros(B, S, H, hd, dtype=torch.bool)
        bad[0, 12, 3] = True
        check({"q": x}, bad)
    x = t["qg"].clone()
    x[1, 39, 1 * 2 * hd + hd + 5] = float("nan")
    bad = torch.zeros(B, S, H, hd, dtype=torch.bool)
    bad[1, 39, 1, 5] = True
    check({"qg": x}, bad)


@pytest.mark.parametrize("splits", [1, 4])
def test_attn_kv8_tiles_outside_the_cache(splits):
    t = _attn_inputs(2, 40, [0, 7], 60, 2, 1, 64, F16, "random")
    clean = _attn(t, 2, 1, 64, long=True, splits=splits)
    bad = dict(t, pos=torch.tensor([-1, 7]))
    got = _attn(bad, 2, 1, 64, long=True, splits=splits)
    assert torch.isnan(got[0]).all() and torch.equal(got[1], clean[1]) and torch.isfinite(clean).all()
    bad = dict(t, parents=t["parents"].clone())
    bad["parents"][1, 39] = 39
    got = _attn(bad, 2, 1, 64, long=True, splits=splits)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], clean[0])


@pytest.mark.parametrize("splits", [1, 4])
def test_attn_kv8_outside_the_cache(splits):
    """Rows whose tokens do not fit, and trees that are none: NaN outputs, caches as they were; the other
    rows of the batch as they are without them."""
    B, S, L, H, G, hd = 3, 5, 40, 2, 1, 64
    t = _attn_inputs(B, S, [35, 0, 7], L, H, G, hd, F16, "random")
    clean = _attn(t, H, G, hd, splits=splits)
    case = (B, S, [35, 0, 7], L, H, G, hd, 16, F16, "random")
    w = list(_write_inputs(case))
    for pos, parents in ((torch.tensor([36, 0, 7]), None), (torch.tensor([-1, 0, 7]), None),
                         (torch.tensor([2 ** 40, 0, 7]), None), (None, (0, 2, 2)), (None, (0, 0, 0)), (None, (0, 3, -2))):
        bad = dict(t)
        wb = list(w)
        if pos is not None:
            bad["pos"] = wb[10] = pos
        else:
            bad["parents"], wb[11] = t["parents"].clone(), w[11].clone()
            bad["parents"][parents[0], parents[1]] = wb[11][parents[0], parents[1]] = parents[2]
        got = _attn(bad, H, G, hd, splits=splits)
        assert torch.isnan(got[0]).all() and torch.equal(got[1:], clean[1:])
        q, caches = _run_write(case, wb)
        assert torch.isnan(q[0]).all() and torch.isfinite(q[1:]).all()
        for c, before in zip(caches, w[6:10]):
            assert torch.equal(c[0], before[0])


def test_attn_kv8_graph_replays():
    """Write and attention captured: replays at later positions, with eager work between them, give the
    eager results; two captured calls on one stream do not share anything."""
    from mlx_gsq_amd.runtime.kernels import kv8
    B, S, L, H, G, hd, rd = 2, 1, 3000, 12, 2, 256, 64
    case = (B, S, [0], L, H, G, hd, rd, F16, None)
    t = [x if x is None else x.cuda() for x in _write_inputs(case)]
    pos = torch.tensor([5, 2000], device="cuda")

    def step(kc, vc, ks, vs, splits):
        q = kv8.kv8_write(*(x.contiguous() for x in t[:3]), t[3], t[4], t[5], kc, vc, ks, vs, pos, heads=H, kv_heads=G,
                          head_dim=hd, rotary_dim=rd, eps=1e-6)
        return kv8.attn_kv8(q, t[0].contiguous(), kc, vc, ks, vs, pos, heads=H, kv_heads=G, head_dim=hd, splits=splits)
    bufs = [x.clone() for x in t[6:10]]
    step(*[x.clone() for x in bufs], 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for splits in (8, 1):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step(*bufs, splits)
            graphs.append((g, out, splits))
    torch.cuda.current_stream().wait_stream(side)
    eager = [x.clone() for x in t[6:10]]
    for i in range(4):
        for g, out, splits in graphs:
            want = step(*eager, splits)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(bufs, eager))
        pos += 17
        t[0].mul_(1.01)


def test_kv8_on_another_stream():
    """Calls follow the current stream's order."""
    from mlx_gsq_amd.runtime.kernels import kv8
    t = _attn_inputs(1, 1, [2000], 2001, 24, 4, 256, F16)
    want = _attn(t, 24, 4, 256)
    d = {n: x.cuda() for n, x in t.items() if x is not None}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            x = (x @ x).clamp_(-1, 1)  # work that the copy below waits for
        q = d["q"] + 0 * x[0, 0].nan_to_num().to(F16)
        got = kv8.attn_kv8(q, d["qg"], d["k"], d["v"], d["ks"], d["vs"], d["pos"], heads=24, kv_heads=4, head_dim=256)
    side.synchronize()
    assert torch.equal(got.cpu(), want)


def test_attn_kv8_past_32_bit_offsets():
    """A cache of more than 2^32 bytes for each of K and V: the last batch row's positions."""
    B, S, L, H, G, hd = 3, 2, 1500000, 6, 4, 256
    H = 24
    t = _attn_inputs(1, S, [300], 310, H, G, hd, F16)
    want, tol = _reference(t, H, G, hd)
    from mlx_gsq_amd.runtime.kernels import kv8
    kc = torch.zeros(B, G, L, hd, dtype=torch.uint8, device="cuda")
    vc, ks = torch.zeros_like(kc), torch.zeros(B, G, L, device="cuda")
    vs = torch.zeros_like(ks)
    assert kc.numel() > 2 ** 32
    for c, n in ((kc, "k"), (vc, "v"), (ks, "ks"), (vs, "vs")):
        c[2, :, :310] = t[n][0].cuda()
    q, qg = (t[n].cuda().expand(B, -1, -1).contiguous() for n in ("q", "qg"))
    got = kv8.attn_kv8(q, qg, kc, vc, ks, vs, torch.tensor([300], device="cuda"), heads=H, kv_heads=G, head_dim=hd)
    _check(got[2:].cpu(), want, tol, F16)
    k, v = kv8.kv8_read(kc, vc, ks, vs, dtype=F16, start=290, length=12)
    assert torch.equal(k[2].cpu(), _values(t["k"], t["ks"])[0, :, 290:302].float().to(F16))
    # and a position past 2^32 / (256 bytes) of one head, written and read back
    big = torch.zeros(1, 1, 17000000, 256, dtype=torch.uint8, device="cuda")
    big_v, sc, sv = torch.zeros_like(big), torch.zeros(1, 1, 17000000, device="cuda"), torch.zeros(1, 1, 17000000, device="cuda")
    case = (1, 2, [16900000], 1, 6, 1, 256, 64, F16, None)
    w = [x if x is None else x.cuda() for x in _write_inputs(case)]
    kv8.kv8_write(*(x.contiguous() for x in w[:3]), w[3], w[4], w[5], big, big_v, sc, sv, w[10], heads=6, kv_heads=1,
                  head_dim=256, rotary_dim=64, eps=1e-6)
    u, s = _quantise(w[2].cpu().double().view(1, 2, 1, 256))
    assert torch.equal(big_v[0, 0, 16900000:16900002].cpu(), u[0, :, 0])
    assert torch.equal(sv[0, 0, 16900000:16900002].cpu(), s[0, :, 0])
    assert int((sv != 0).sum()) == 2 and int(big_v[0, 0, :16900000:4099].any()) == 0


def test_kv8_empty_calls():
    from mlx_gsq_amd.runtime.kernels import kv8
    for B, S in ((0, 3), (2, 0)):
        t = _attn_inputs(max(B, 1), max(S, 1), [0], 8, 4, 2, 64, F16)
        d = {n: x.cuda() for n, x in t.items() if x is not None}
        out = kv8.attn_kv8(d["q"][:B, :S], d["qg"][:B, :S], d["k"][:B], d["v"][:B], d["ks"][:B], d["vs"][:B], d["pos"], heads=4,
                           kv_heads=2, head_dim=64)
        assert out.shape == (B, S, 256)


@pytest.mark.parametrize("long", [False, True])
def test_attn_kv8_outputs_are_not_shifted(long):
    """Averages over thousands of positions, far smaller than the values, whose sizes vary: what the float32 sums
    leave in all dims alike is within one float32 rounding of the rows' largest values (2^-24 times their
    weighted mean)."""
    B, S, pos, L, H, G, hd = 1, 24, [8000], 8024, 64, 8, 256
    t = _attn_inputs(B, S, pos, L, H, G, hd, F16)
    t["qg"].view(B, S, H, 2 * hd)[..., hd:] = 60.0  # gates of 1
    got = _attn(t, H, G, hd, long=long).double().view(B, S, H, hd)
    want, _ = _reference(t, H, G, hd)
    largest = torch.empty(B, S, H, 1, dtype=torch.float64)
    see = torch.arange(L)[None, :] <= pos[0] + torch.arange(S)[:, None]
    for h in range(H):
        k, q = _values(t["k"][0, h // 8], t["ks"][0, h // 8]), t["q"][0].double().view(S, H, hd)[:, h]
        p = torch.softmax((torch.matmul(q, k.t().contiguous()) * hd ** -0.5).masked_fill(~see, float("-inf")), -1)
        largest[0, :, h, 0] = 127 * torch.matmul(p, t["vs"][0, h // 8].double())
    # the rounding to fp16 has no direction: of B S H hd outputs, each off by 2^-11 / sqrt(3) of itself at most (root
    # mean square), it leaves this in the mean (4 sigma)
    noise = 4 * float((want / largest).square().mean().sqrt()) * 2.0 ** -11 / math.sqrt(3 * want.numel())
    assert noise < 2.0 ** -25
    assert abs(float(((got - want) / largest).mean())) <= 2.0 ** -24 + noise


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attn_kv8_outputs_are_rounded_once(dtype, long):
    """Scores, weights and sums as float32 has them: an output differs from the rounded float64 value only where that
    lies within eight float32 roundings of the rows' largest values (2^-24 times their weighted mean) of a border."""
    B, S, pos, L, H, G, hd = 2, 12, [300, 211], 312, 24, 4, 128
    t = _attn_inputs(B, S, pos, L, H, G, hd, dtype)
    t["qg"].view(B, S, H, 2 * hd)[..., hd:] = 60.0  # gates of 1
    got = _attn(t, H, G, hd, long=long).view(B, S, H, hd)
    want, _ = _reference(t, H, G, hd)
    off = torch.empty(B, S, H, 1, dtype=torch.float64)
    for b in range(B):
        n = pos[b] + S
        see = torch.arange(n)[None, :] <= pos[b] + torch.arange(S)[:, None]
        for h in range(H):
            k, q = _values(t["k"][b, h // 6, :n], t["ks"][b, h // 6, :n]), t["q"][b].double().view(S, H, hd)[:, h]
            p = torch.softmax((torch.matmul(q, k.t().contiguous()) * hd ** -0.5).masked_fill(~see, float("-inf")), -1)
            off[b, :, h, 0] = 8 * 2.0 ** -24 * 127 * torch.matmul(p, t["vs"][b, h // 6, :n].double())
    step = torch.finfo(dtype).eps * 2.0 ** want.abs().clamp(min=2.0 ** -14).log2().floor()
    near = (2 * off / step).clamp(max=1.0).sum()  # borders lie a step apart
    assert int((got != want.to(dtype)).sum()) <= float(near)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("long", [False, True])
def test_attn_kv8_values_next_to_the_largest(long, splits):
    """bf16 V rows of up to 127 x 2^121, next to float32's largest number, which any sum of two of them passes:
    their averages are finite."""
    B, S, pos, L, H, G, hd = 1, 24, [350], 374, 4, 2, 64
    t = _attn_inputs(B, S, pos, L, H, G, hd, BF16)
    t["vs"] = 0.25 + 0.75 * t["vs"] / t["vs"].amax()
    want, tol = _reference(t, H, G, hd)
    t["vs"] = t["vs"] * 2.0 ** 121
    got = _attn(t, H, G, hd, long=long, splits=splits)
    _check(got.double() * 2.0 ** -121, want, tol, BF16)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("long", [False, True])
def test_attn_kv8_scores_below_the_range(long, splits):
    """A row whose scores all pass float32's range downwards has no weights: NaN, as their softmax gives; the
    other rows are what they are without it."""
    B, S, pos, L, H, G, hd = 1, 40, [300], 340, 4, 2, 64
    t = _attn_inputs(B, S, pos, L, H, G, hd, BF16)
    t["k"], t["ks"] = _quantise(_values(t["k"], t["ks"]).abs() + 1)
    clean, tol = _reference(t, H, G, hd)
    q = t["q"].view(B, S, H, hd)
    q[0, 12, 1] = -3e38
    got = _attn(t, H, G, hd, long=long, splits=splits).view(B, S, H, hd)
    assert torch.isnan(got[0, 12, 1]).all()
    keep = torch.ones(B, S, H, dtype=torch.bool)
    keep[0, 12, 1] = False
    _check(got[keep], clean[keep], tol[keep], BF16)
