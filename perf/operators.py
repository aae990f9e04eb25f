"""Performance cases of the operators around an 8-bit attention cache and trees of drafted tokens.

Kinds (sizes of the 27B hybrid decoder unless a case says otherwise: 24 query heads over 4 KV heads
of 256, 64 rotated dims; GatedDeltaNet of 48 value and 16 key heads of 128, convolution kernel 4):

* ``kv8``: s new tokens of b rows behind ``pos`` cached ones: q and k normalized and rotated, k and v
  quantised into the cache (``kv8_write``), and the cache read back as 16-bit rows (``kv8_read``).
* ``attn``: attention of s new tokens over the 8-bit cache (``attn_kv8``): one token (decoding) or a
  prompt; ``ragged``: rows of a batch at positions of their own.
* ``tree``: the same for a tree of s drafted tokens (a token sees the cache and its ancestors).
* ``gdn``: the GatedDeltaNet over a tree of s drafted tokens (``gdn_tree``).

The plain forms are elementary torch operations in 32 bits; ``exact`` goes by the definitions in
64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "mlx-gsq-rco_amd")
if _PKG not in sys.path:
    sys.path.insert(1, _PKG)

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS, THETA, CONV = 1e-6, 1e7, 4


# ---- the cases ---------------------------------------------------------------------------

def _attn(kind, b, s, pos, dtype, heads=24, kv_heads=4, hd=256, rd=64, ragged=False, **kw):
    return dict({"kind": kind, "b": b, "s": s, "pos": pos, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
                 "hd": hd, "rd": rd, "ragged": ragged}, **kw)


def _gdn(b, s, dtype, hk=16, hv=48, dk=128, dv=128):
    return {"kind": "gdn", "b": b, "s": s, "dtype": dtype, "hk": hk, "hv": hv, "dk": dk, "dv": dv}


def listed():
    return [
        # a decoding step of a small batch, and a prompt, written to the cache and handed to 16-bit code
        dict(_attn("kv8", 8, 1, 511, "bf16"), name="kv8_step_8rows"),
        dict(_attn("kv8", 1, 2047, 0, "fp16"), name="kv8_prompt_2047"),
        # single tokens: a chat's short context, one long document, a serving batch at its rows' own lengths
        dict(_attn("attn", 1, 1, 300, "fp16"), name="attn_step_short"),
        dict(_attn("attn", 1, 1, 131071, "fp16"), name="attn_step_long"),
        dict(_attn("attn", 32, 1, 8191, "bf16", ragged=True), name="attn_step_32rows"),
        # prompts: a short odd one, a long one, a turn that continues a cached conversation (head dim 128)
        dict(_attn("attn", 1, 333, 0, "bf16"), name="attn_prompt_333"),
        dict(_attn("attn", 1, 4096, 0, "fp16"), name="attn_prompt_4096"),
        dict(_attn("attn", 2, 700, 5000, "bf16", 32, 8, 128, 128), name="attn_turn_700"),
        # drafted trees: a small one over a chat, a wide one for a batch over long contexts
        dict(_attn("tree", 1, 13, 2000, "fp16"), name="tree_13"),
        dict(_attn("tree", 4, 64, 16000, "bf16", ragged=True), name="tree_64_4rows"),
        # the recurrent layer of the same trees
        dict(_gdn(1, 13, "fp16"), name="gdn_tree_13"),
        dict(_gdn(4, 64, "bf16"), name="gdn_tree_64_4rows"),
    ]


MAX_FLOPS = 2.1e11   # of the largest listed prompt
MAX_CACHE = 131072   # positions over all rows


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["kv8", "step", "step", "prompt", "prompt", "tree", "tree", "gdn"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "gdn":
        hk = rng.choice([2, 4, 16])
        return _gdn(_log(rng, 1, 4), _log(rng, 1, 64), dtype, hk, hk * rng.choice([1, 2, 3]), rng.choice([64, 128]),
                    rng.choice([64, 128]))
    hd = rng.choice([64, 128, 256, 256])
    kv_heads = rng.choice([1, 2, 4, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 6, 6, 8])
    rd = rng.choice([hd // 4, hd // 2, hd])
    b = rng.choice([1, 1, _log(rng, 1, 32)])
    ragged = b > 1 and rng.random() < 0.6
    room = MAX_CACHE * 4 // max(4, kv_heads) // b
    if kind == "kv8":
        room = min(room, 16384 // b)
        s = rng.choice([1, _log(rng, 1, 2047)])
        s = min(s, room)
        return _attn(kind, b, s, _log(rng, 1, max(1, room - s)) - 1, dtype, heads, kv_heads, hd, rd, ragged)
    if kind == "step":
        return _attn("attn", b, 1, _log(rng, 1, room) - 1, dtype, heads, kv_heads, hd, rd, ragged)
    if kind == "tree":
        s = _log(rng, 2, 64)
        return _attn("tree", b, s, _log(rng, 1, min(room, 20000)) - 1, dtype, heads, kv_heads, hd, rd, ragged)
    b = rng.choice([1, 1, 2, 3])
    while True:
        case = _attn("attn", b, _log(rng, 2, 4096), rng.choice([0, _log(rng, 1, 8192)]), dtype, heads, kv_heads, hd, rd,
                     b > 1 and ragged)
        # the plain form's scores over every position, in 32 bits, within those of the largest listed case
        if (case["s"] * (case["s"] + case["pos"]) * heads * b <= 4096 * 4096 * 24 and work(case)["flops"] <= MAX_FLOPS):
            return case


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=torch.device("cuda", torch.cuda.current_device())).manual_seed(int(seed))


def _positions(case):
    """Cached tokens of each row: all ``pos``, or (ragged) falling from it to about a half."""
    return [case["pos"] - (case["pos"] * i // (2 * case["b"]) if case["ragged"] else 0) for i in range(case["b"])]


def _parents(b, s, gen):
    """A random tree for each row: a node's parent is one of the few drafted before it, or the cache's
    last token (-1)."""
    back = 1 + (torch.rand(b, s, device=gen.device, generator=gen) ** 2 * 6).long()
    return (torch.arange(s, device=gen.device) - back).clamp(min=-1).to(torch.int32)


def _quantise(x):
    """8-bit rows of x as a cache holds them: (values + 128 as bytes, scale of each row)."""
    scale = x.abs().amax(-1) / 127
    return ((x / scale[..., None]).round() + 128).to(torch.uint8), scale


def prepare(case, seed):
    gen = _gen(seed)
    dev, dt = gen.device, DTYPES[case["dtype"]]
    b, s = case["b"], case["s"]

    def rnd(*shape):
        return torch.randn(*shape, device=dev, generator=gen)
    st = {"case": case}
    if case["kind"] == "gdn":
        hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "dk", "dv"))
        conv_dim = 2 * hk * dk + hv * dv
        qkvz = rnd(b, s, conv_dim + hv * dv).to(dt)
        st["qkv"], st["z"] = qkvz[..., :conv_dim], qkvz[..., conv_dim:]
        st["ab"] = rnd(b, s, 2 * hv).to(dt)
        st["conv_state"], st["conv_w"] = rnd(b, CONV - 1, conv_dim).to(dt), (0.5 * rnd(conv_dim, CONV)).to(dt)
        # A in [1, 16] and softplus(dt_bias) in [0.001, 0.1]: the architecture's initial range
        st["ssm_a"] = -torch.exp(torch.rand(hv, device=dev, generator=gen) * math.log(16.0))
        dt_ = torch.exp(torch.rand(hv, device=dev, generator=gen) * math.log(100.0) + math.log(0.001))
        st["dt_bias"] = torch.log(torch.expm1(dt_))
        st["rec"] = 0.1 * rnd(b, hv, dk, dv)
        st["norm_w"] = (1 + 0.1 * rnd(dv)).to(dt)
        st["parents"] = _parents(b, s, gen)
        return st
    H, G, hd, rd = case["heads"], case["kv_heads"], case["hd"], case["rd"]
    pos = _positions(case)
    L = max(pos) + s
    st["pos"] = torch.tensor(pos if case["ragged"] else pos[:1], device=dev)
    st["qg"] = rnd(b, s, H * 2 * hd).to(dt)
    # cached rows: keys with a part common to a head's (attention sinks), values of varying size by token
    common = 0.5 * rnd(G, 1, hd)
    k, ks = zip(*(_quantise(rnd(G, L, hd) + common) for _ in range(b)))
    v, vs = zip(*(_quantise(rnd(G, L, hd) * torch.exp(0.5 * rnd(G, L, 1))) for _ in range(b)))
    st["k"], st["ks"], st["v"], st["vs"] = (torch.stack(t) for t in (k, ks, v, vs))
    if case["kind"] == "kv8":
        st["kn"], st["vn"] = rnd(b, s, G * hd).to(dt), rnd(b, s, G * hd).to(dt)
        st["qw"], st["kw"] = (1 + 0.1 * rnd(hd)).to(dt), (1 + 0.1 * rnd(hd)).to(dt)
        st["freq"] = 1.0 / THETA ** (torch.arange(0, rd, 2, dtype=torch.float64, device=dev) / rd)
        return st
    q = rnd(b, s, G, H // G, hd) + common.view(G, 1, hd)
    st["q"] = q.reshape(b, s, H * hd).to(dt)
    st["parents"] = _parents(b, s, gen) if case["kind"] == "tree" else None
    return st


# ---- one pass ----------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["kind"] == "gdn":
        return _run_gdn(state)
    if case["kind"] == "kv8":
        return _run_kv8(state)
    return _run_attn(state)


def _run_kv8(s):
    c = s["case"]
    if own:
        from mlx_gsq_amd.runtime.kernels import kv8
        q = kv8.kv8_write(s["qg"], s["kn"], s["vn"], s["qw"], s["kw"], s["freq"], s["k"], s["v"], s["ks"], s["vs"],
                          s["pos"], heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["hd"], rotary_dim=c["rd"], eps=EPS)
        k, v = kv8.kv8_read(s["k"], s["v"], s["ks"], s["vs"], dtype=s["qg"].dtype)
        return {"q": q, "k": k, "v": v}
    B, S, H, G, hd, rd, dt = c["b"], c["s"], c["heads"], c["kv_heads"], c["hd"], c["rd"], s["qg"].dtype
    at = s["pos"].expand(B)[:, None] + torch.arange(S, device=s["pos"].device)  # (B, S)
    ang = at.double()[..., None, None] * s["freq"]
    cos, sin = ang.cos(), ang.sin()

    def norm_rope(x, w):  # in 64 bits: rounding to 8 bits jumps at values next to a border
        x = x.double()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
        lo, hi = x[..., :rd // 2], x[..., rd // 2:rd]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., rd:]], -1)
    q = norm_rope(s["qg"].reshape(B, S, H, 2 * hd)[..., :hd], s["qw"])
    row = torch.arange(B, device=at.device)[:, None]
    for name, x in (("k", norm_rope(s["kn"].reshape(B, S, G, hd), s["kw"])), ("v", s["vn"].double().reshape(B, S, G, hd))):
        scale = (x.abs().amax(-1) / 127).float()
        u = torch.where(scale[..., None] > 0, x / scale[..., None].double(), 0.0).round() + 128
        s[name][row, :, at] = u.to(torch.uint8)
        s[name + "s"][row, :, at] = scale
    k, v = (((s[n].float() - 128) * s[n + "s"][..., None]).to(dt) for n in ("k", "v"))
    return {"q": q.reshape(B, S, H * hd).to(dt), "k": k, "v": v}


def _ancestors(parents):
    """(B, S, S) truth values: node j is node i or one of its ancestors."""
    n = parents.shape[1]
    up = (parents[..., None] == torch.arange(n, device=parents.device)).float() + torch.eye(n, device=parents.device)
    for _ in range(6):  # paths of up to 64 steps
        up = torch.matmul(up, up.contiguous()).clamp(max=1)
    return up > 0


def _visible(pos, S, L, parents):
    """(B or 1, S, L): the positions that each new token attends to."""
    key = torch.arange(L, device=pos.device)
    if parents is None:
        return key <= (pos[:, None] + torch.arange(S, device=pos.device))[..., None]
    B = parents.shape[0]
    drafted = key - pos.expand(B)[:, None]  # (B, L): node of each position
    seen = torch.gather(_ancestors(parents), 2, drafted.clamp(0, S - 1)[:, None].expand(B, S, L))
    return torch.where(((drafted >= 0) & (drafted < S))[:, None], seen, (drafted < 0)[:, None])


def _run_attn(s):
    c = s["case"]
    if own:
        from mlx_gsq_amd.runtime.kernels import kv8
        return kv8.attn_kv8(s["q"], s["qg"], s["k"], s["v"], s["ks"], s["vs"], s["pos"], heads=c["heads"],
                            kv_heads=c["kv_heads"], head_dim=c["hd"], parents=s["parents"])
    B, S, H, G, hd = c["b"], c["s"], c["heads"], c["kv_heads"], c["hd"]
    L = s["k"].shape[2]
    k = (s["k"].float() - 128) * s["ks"][..., None]
    q = s["q"].float().reshape(B, S, G, H // G, hd).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * S, hd)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, G, H // G, S, L) * hd ** -0.5
    scores.masked_fill_(~_visible(s["pos"], S, L, s["parents"])[:, None, None], float("-inf"))
    p = (scores - scores.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    v = (s["v"].float() - 128) * s["vs"][..., None]
    o = torch.matmul(p.view(B, G, -1, L), v).view(B, H, S, hd).transpose(1, 2)
    gate = s["qg"].reshape(B, S, H, 2 * hd)[..., hd:].float()
    return (o / (1 + torch.exp(-gate))).reshape(B, S, H * hd).to(s["q"].dtype)


def _run_gdn(s):
    c = s["case"]
    hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
    if own:
        from mlx_gsq_amd.runtime.kernels import model_ops
        return model_ops.gdn_tree(s["qkv"], s["z"], s["ab"], s["conv_state"], s["conv_w"], s["ssm_a"], s["dt_bias"],
                                  s["rec"], s["norm_w"], s["parents"], key_heads=hk, value_heads=hv, head_k_dim=dk,
                                  head_v_dim=dv, eps=EPS)
    B, S, dt = c["b"], c["s"], s["qkv"].dtype
    # window of a node: its ancestors' inputs, then the state's (parent of -1: the state's last, -2, ..)
    rows = torch.cat([s["conv_state"], s["qkv"]], 1).float()  # node i at CONV - 1 + i
    up = torch.cat([torch.arange(-1, CONV - 2, device=rows.device).expand(B, -1), s["parents"].long() + CONV - 1], 1).clamp(min=0)
    at = torch.arange(S, device=rows.device).expand(B, S) + CONV - 1
    acc = 0.0
    for j in range(CONV - 1, -1, -1):
        acc = acc + torch.gather(rows, 1, at[..., None].expand(-1, -1, rows.shape[2])) * s["conv_w"].float()[:, j]
        at = torch.gather(up, 1, at)
    x = acc / (1 + torch.exp(-acc))
    q, k, v = x.split([hk * dk, hk * dk, hv * dv], -1)

    def heads(t, size):  # per value head h the normalized rows of key head h % hk
        t = t.reshape(B, S, hk, dk)
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * size
        return t.repeat(1, 1, hv // hk, 1).transpose(1, 2)
    q, k, v = heads(q, 1 / dk), heads(k, dk ** -0.5), v.reshape(B, S, hv, dv).transpose(1, 2)
    a, b = s["ab"].float().split(hv, -1)
    beta = (1 / (1 + torch.exp(-b))).transpose(1, 2)[..., None]                       # (B, hv, S, 1)
    a = a + s["dt_bias"]
    log_decay = s["ssm_a"] * torch.where(a > 20, a, torch.log1p(torch.exp(a.clamp(max=20))))
    path = _ancestors(s["parents"])                                                   # (B, S, S)
    g = torch.matmul(path.float(), log_decay).transpose(1, 2)                         # (B, hv, S): along the path
    ratio = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(~path[:, None], float("-inf")))
    grown = torch.exp(g)[..., None]
    kt = k.transpose(2, 3).contiguous()
    eye = torch.eye(S, device=rows.device)
    m = beta * ratio * torch.matmul(k, kt) * (1 - eye)
    u = beta * (v - grown * torch.matmul(k, s["rec"]))
    for _ in range(6):  # (1 + m)^-1 = (1 - m)(1 + m^2)(1 + m^4) ..: no path is longer than 64
        u = u - torch.matmul(m, u) if _ == 0 else u + torch.matmul(m, u)
        m = torch.matmul(m, m.contiguous())
    o = grown * torch.matmul(q, s["rec"]) + torch.matmul(ratio * torch.matmul(q, kt), u)
    o = o.transpose(1, 2)                                                             # (B, S, hv, dv)
    o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * s["norm_w"].float()
    z = s["z"].float().reshape(B, S, hv, dv)
    return (o * z / (1 + torch.exp(-z))).reshape(B, S, hv * dv).to(dt)


# ---- what a pass cannot do without -------------------------------------------------------

def work(case):
    b, s = case["b"], case["s"]
    if case["kind"] == "gdn":
        hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "dk", "dv"))
        conv_dim = 2 * hk * dk + hv * dv
        rows = 2 * b * s * (conv_dim + 2 * hv * dv + 2 * hv)
        weights = 2 * conv_dim * CONV + 2 * b * (CONV - 1) * conv_dim + 2 * dv + 8 * hv + 4 * b * s
        # two products with the state, and the tree's with a few ancestors to a node
        return {"bytes": rows + weights + 4 * b * hv * dk * dv,
                "flops": b * s * (hv * (4.0 * dk * dv + 8 * 4 * (dk + dv)) + 2.0 * CONV * conv_dim)}
    H, G, hd = case["heads"], case["kv_heads"], case["hd"]
    pos = _positions(case)
    if case["kind"] == "kv8":
        new = b * s * (2 * H * hd * 2 + 2 * G * hd * 2 + 2 * G * (hd + 4)) + 4 * hd + 4 * case["rd"]
        L = max(pos) + s
        return {"bytes": new + b * L * G * 2 * (hd + 4 + 2 * hd), "flops": 10.0 * b * s * (H + 2 * G) * hd + 2.0 * b * L * G * 2 * hd}
    cached = sum(p + s for p in pos)
    if case["kind"] == "tree":
        seen = sum(s * (p + 5) for p in pos)  # the cache, itself and a few ancestors
    else:
        seen = sum(s * p + s * (s + 1) // 2 for p in pos)
    return {"bytes": cached * G * 2 * (hd + 4) + b * s * H * hd * 2 * 3, "flops": 4.0 * H * hd * seen}


# ---- the definitions in 64 bits ----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"gdn": _exact_gdn, "kv8": _exact_kv8}.get(case["kind"], _exact_attn)(s)


def _exact_kv8(s):
    c = s["case"]
    B, S, H, G, hd, half = c["b"], c["s"], c["heads"], c["kv_heads"], c["hd"], c["rd"] // 2
    pos = s["pos"].expand(B).tolist()

    def turned(x, w, p):  # x (S, n, hd) at positions p ..
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
        z = torch.polar(torch.ones(S, half, dtype=torch.float64, device=x.device),
                        torch.arange(p, p + S, device=x.device).double()[:, None] * s["freq"])[:, None]
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)
    caches = {n: (s[n].double() - 128) * s[n + "s"].double()[..., None] for n in ("k", "v")}
    q = []
    for i in range(B):
        q.append(turned(s["qg"][i].reshape(S, H, 2 * hd)[..., :hd], s["qw"], pos[i]).reshape(S, H * hd))
        new = {"k": turned(s["kn"][i].reshape(S, G, hd), s["kw"], pos[i]), "v": s["vn"][i].double().reshape(S, G, hd)}
        for n, x in new.items():
            step = (x.abs().amax(-1, keepdim=True) / 127).float().double()  # the scale is held in 32 bits
            caches[n][i, :, pos[i]:pos[i] + S] = ((x / step).round() * step).transpose(0, 1)
    return {"q": torch.stack(q), "k": caches["k"], "v": caches["v"]}


def _exact_attn(s):
    c = s["case"]
    B, S, H, G, hd = c["b"], c["s"], c["heads"], c["kv_heads"], c["hd"]
    pos = s["pos"].expand(B).tolist()
    out = torch.empty(B, S, H, hd, dtype=torch.float64, device=s["q"].device)
    for i in range(B):
        n = pos[i] + S
        later = torch.ones(S, S, dtype=torch.bool, device=out.device).triu(1)
        if s["parents"] is not None:
            later = torch.ones_like(later)
            up = s["parents"][i].tolist()
            for t in range(S):
                if up[t] >= 0:
                    later[t] = later[up[t]]
                later[t, t] = False
        for h in range(H):
            g = h // (H // G)
            k = (s["k"][i, g, :n].double() - 128) * s["ks"][i, g, :n, None].double()
            v = (s["v"][i, g, :n].double() - 128) * s["vs"][i, g, :n, None].double()
            a = torch.mm(s["q"][i].view(S, H, hd)[:, h].double(), k.t().contiguous()) / math.sqrt(hd)
            a[:, pos[i]:][later] = -math.inf
            out[i, :, h] = torch.mm((a - torch.logsumexp(a, -1, keepdim=True)).exp(), v)
    gate = s["qg"].view(B, S, H, 2 * hd)[..., hd:].double()
    return (out * torch.sigmoid(gate)).reshape(B, S, H * hd)


def _exact_gdn(s):
    c = s["case"]
    hk, hv, dk, dv, B, S = c["hk"], c["hv"], c["dk"], c["dv"], c["b"], c["s"]
    out = torch.empty(B, S, hv, dv, dtype=torch.float64, device=s["rec"].device)
    w, first = s["conv_w"].double(), s["conv_state"].double()
    head = torch.arange(hv, device=out.device) % hk
    for i in range(B):
        states, windows = {-1: s["rec"][i].double()}, {-1: first[i]}
        for t, p in enumerate(s["parents"][i].tolist()):
            win = torch.cat([windows[p], s["qkv"][i, t].double()[None]])
            windows[t] = win[1:]
            x = (win * w.t()).sum(0)
            q, k, v = (x * torch.sigmoid(x)).split([hk * dk, hk * dk, hv * dv])
            q, k = (y.view(hk, dk) / (y.view(hk, dk).pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() for y in (q, k))
            q, k, v = q[head] / dk, k[head] / math.sqrt(dk), v.view(hv, dv)
            a, b = s["ab"][i, t].double().split(hv)
            decay = torch.exp(s["ssm_a"].double() * torch.nn.functional.softplus(a + s["dt_bias"].double()))
            st = states[p] * decay[:, None, None]
            read = (st * k[..., None]).sum(1)
            states[t] = st + k[..., None] * (torch.sigmoid(b)[:, None] * (v - read))[:, None]
            y = (states[t] * q[..., None]).sum(1)
            y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["norm_w"].double()
            z = s["z"][i, t].double().view(hv, dv)
            out[i, t] = y * z * torch.sigmoid(z)
    return out.view(B, S, hv * dv)
