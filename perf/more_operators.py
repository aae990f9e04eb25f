"""Performance cases of the operators that serve many requests in one step: their tokens packed behind one
another, K and V in pages that are handed out on the GPU.

Kinds (sizes of the 27B hybrid decoder unless a case says otherwise: 24 query heads over 4 KV heads of 256, 64 rotated
dims; GatedDeltaNet of 48 value and 16 key heads of 128, convolution kernel 4):

* ``plan``: the step's layout from the requests' lengths: pages taken, block table, slots and positions
  (``page_plan``); the prompts of the step end with it and give their pages back (``page_release``).
* ``write``: q and k normalized per head and rotated, k and v written to their slots (``paged_write``).
* ``attn``: attention of the packed tokens over their requests' pages (``attn_paged``).
* ``gdn``: the GatedDeltaNet over the packed tokens, each request with states of its own (``gdn_packed``).

A step holds ``b`` sequences: the first ``prompts`` of them bring ``new`` tokens falling to about half of that
behind ``ppos`` cached ones, the others one token each behind ``pos`` falling to about half.

The plain forms are elementary torch operations in 32 bits; ``exact`` goes by the definitions in 64 bits.
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
EPS, THETA, CONV, CHUNK = 1e-6, 1e7, 4, 64


# ---- the cases ---------------------------------------------------------------------------

def _step(kind, b, prompts=0, new=1, ppos=0, pos=0, **kw):
    return dict({"kind": kind, "b": b, "prompts": prompts, "new": new, "ppos": ppos, "pos": pos}, **kw)


def _attn(kind, dtype, b, prompts=0, new=1, ppos=0, pos=0, heads=24, kv_heads=4, hd=256, rd=64, page=64):
    return _step(kind, b, prompts, new, ppos, pos, dtype=dtype, heads=heads, kv_heads=kv_heads, hd=hd, rd=rd, page=page)


def _gdn(dtype, b, prompts=0, new=1, ppos=0, hk=16, hv=48, dk=128, dv=128):
    return _step("gdn", b, prompts, new, ppos, 100, dtype=dtype, hk=hk, hv=hv, dk=dk, dv=dv)


def listed():
    return [
        # a decoding step of a small batch; a busy server's step, four long prompts beside 250 running requests
        dict(_step("plan", 16, pos=2000, page=64), name="plan_step_16"),
        dict(_step("plan", 254, 4, 8191, 0, 9000, page=16), name="plan_mixed_254"),
        # a decoding step of eight requests; five prompts of odd lengths
        dict(_attn("write", "bf16", 8, pos=511), name="write_step_8"),
        dict(_attn("write", "fp16", 5, 5, 1111, page=16), name="write_prompts_5"),
        # single tokens: a chat's short context, one long document, a serving batch of all lengths
        dict(_attn("attn", "fp16", 1, pos=300, page=16), name="attn_step_short"),
        dict(_attn("attn", "fp16", 1, pos=131071), name="attn_step_long"),
        dict(_attn("attn", "bf16", 32, pos=16383), name="attn_step_32"),
        # whole prompts packed behind one another (head dim 128); a chunk of a long document beside running requests
        dict(_attn("attn", "bf16", 5, 5, 2001, heads=32, kv_heads=8, hd=128, rd=128, page=16), name="attn_prompts_5"),
        dict(_attn("attn", "fp16", 24, 1, 1024, 30000, 4000), name="attn_chunk_24"),
        # the recurrent layer of a decoding step, of a short turn beside running requests, and of long prompts
        dict(_gdn("bf16", 32), name="gdn_step_32"),
        dict(_gdn("fp16", 9, 1, 61, 1000), name="gdn_turn_61"),
        dict(_gdn("bf16", 3, 3, 2047), name="gdn_prompts_3"),
    ]


MAX_FLOPS = 8.5e11    # of the largest listed attention
MAX_SCORES = 8e8      # of the plain form's float32 scores
MAX_CACHE = 600000    # positions x KV heads over all rows of the plain form's float32 caches, at head dim 256


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "write", "step", "step", "step", "prompt", "prompt", "prompt", "gdn", "gdn"])
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        b = _log(rng, 1, 250)
        return _step("plan", b, rng.randint(0, min(b, 4)), _log(rng, 2, 8191), 0, _log(rng, 1, 9000), page=page)
    if kind == "gdn":
        hk = rng.choice([2, 4, 16])
        heads = (hk, hk * rng.choice([1, 2, 3]), rng.choice([64, 128]), rng.choice([64, 128]))
        if rng.random() < 0.3:
            return _gdn(dtype, _log(rng, 1, 32), 0, 1, 0, *heads)
        prompts = rng.randint(1, 3)
        return _gdn(dtype, prompts + rng.choice([0, _log(rng, 1, 16)]), prompts, _log(rng, 2, 2047),
                    rng.choice([0, _log(rng, 1, 5000)]), *heads)
    hd = rng.choice([64, 128, 256, 256])
    kv_heads = rng.choice([1, 2, 4, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 6, 6, 8])
    rd = rng.choice([hd // 4, hd // 2, hd])
    if kind == "write":
        prompts = rng.randint(0, 5)
        return _attn("write", dtype, prompts + _log(rng, 1, 32), prompts, _log(rng, 2, 1111), 0, _log(rng, 1, 4000) - 1, heads,
                     kv_heads, hd, rd, page)
    while True:
        if kind == "step":
            case = _attn("attn", dtype, _log(rng, 1, 64), 0, 1, 0, _log(rng, 1, 131072) - 1, heads, kv_heads, hd, rd, page)
        else:
            prompts = rng.randint(1, 5)
            case = _attn("attn", dtype, prompts + rng.choice([0, _log(rng, 1, 23)]), prompts, _log(rng, 2, 2001),
                         rng.choice([0, _log(rng, 1, 30000)]), _log(rng, 1, 4000) - 1, heads, kv_heads, hd, rd, page)
        p, s, m = case["prompts"], case["new"], case["b"] - case["prompts"]
        cache = max(p * (case["ppos"] + s), m * (case["pos"] + 1)) * kv_heads
        if cache <= MAX_CACHE * 4 and p * heads * s * (case["ppos"] + s) <= MAX_SCORES and work(case)["flops"] <= MAX_FLOPS:
            return case


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=torch.device("cuda", torch.cuda.current_device())).manual_seed(int(seed))


def _lengths(case):
    """(cached tokens, new tokens) of each sequence of the step."""
    p, m = case["prompts"], case["b"] - case["prompts"]
    new = [case["new"] - case["new"] * i // (2 * p) for i in range(p)] + [1] * m
    cached = [case["ppos"] - case["ppos"] * i // (2 * p) for i in range(p)] + [case["pos"] - case["pos"] * i // (2 * m)
                                                                               for i in range(m)]
    return cached, new


def _pages(lengths, page):
    return [-(-n // page) for n in lengths]


def _layout(case, dev, gen, page):
    """A step as its plan says it, over pages in random order: (block table, plan), the plan being (start of each
    sequence, its request, its length, position of each token, slot of each token)."""
    cached, new = _lengths(case)
    total = [c + n for c, n in zip(cached, new)]
    b, need = case["b"], _pages(total, page)
    pages = torch.randperm(sum(need), device=dev, generator=gen).to(torch.int32)
    table = torch.full((b + 2, max(need)), -1, dtype=torch.int32, device=dev)
    rows = torch.randperm(b + 2, device=dev, generator=gen)[:b]
    i32 = dict(dtype=torch.int32, device=dev)
    first = torch.tensor(need, device=dev).cumsum(0) - torch.tensor(need, device=dev)
    of = torch.arange(max(need), device=dev)
    have = torch.tensor(need, device=dev)[:, None] > of
    table[rows] = torch.where(have, pages[(first[:, None] + of).clamp(max=sum(need) - 1)], -1)
    n = torch.tensor(new, device=dev)
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    seq = torch.repeat_interleave(torch.arange(b, device=dev), n)
    pos = torch.tensor(cached, device=dev)[seq] + torch.arange(sum(new), device=dev) - cu[seq]
    slots = table[rows[seq], pos // page].long() * page + pos % page
    return table, (cu.int(), rows.int(), torch.tensor(total, **i32), pos, slots), sum(need)


def prepare(case, seed):
    gen = _gen(seed)
    dev = gen.device

    def rnd(*shape):
        return torch.randn(*shape, device=dev, generator=gen)
    st = {"case": case}
    cached, new = _lengths(case)
    N, b = sum(new), case["b"]
    if case["kind"] == "plan":
        # more requests than the step serves, the pages of the running ones handed out in random order
        page, R = case["page"], b + 6
        held = _pages(cached, page)
        width = max(_pages([c + n for c, n in zip(cached, new)], page)) + 3
        spare = sum(_pages([c + n for c, n in zip(cached, new)], page)) + 5 - sum(held)
        order = torch.randperm(sum(held) + spare, device=dev, generator=gen).to(torch.int32)
        rows = torch.randperm(R, device=dev, generator=gen)[:b]
        st["table"] = torch.full((R, width), -1, dtype=torch.int32, device=dev)
        h = torch.tensor(held, device=dev)
        of = torch.arange(width, device=dev)
        at = spare + (h.cumsum(0) - h)[:, None] + of
        st["table"][rows] = torch.where(h[:, None] > of, order[at.clamp(max=order.numel() - 1)], -1)
        st["free"] = torch.cat([order[:spare], torch.full((sum(held),), -1, dtype=torch.int32, device=dev)])
        st["n_free"] = torch.tensor([spare], dtype=torch.int32, device=dev)
        st["held"], st["lengths"] = (torch.zeros(R, dtype=torch.int32, device=dev) for _ in range(2))
        st["held"][rows] = h.int()
        st["lengths"][rows] = torch.tensor(cached, dtype=torch.int32, device=dev)
        st["requests"], st["new"], st["tokens"] = rows.int(), torch.tensor(new, dtype=torch.int32, device=dev), N
        return st
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "gdn":
        hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "dk", "dv"))
        conv_dim = 2 * hk * dk + hv * dv
        st["plan"] = _layout(case, dev, gen, 64)[1]
        qkvz = rnd(N, conv_dim + hv * dv).to(dt)
        st["qkv"], st["z"] = qkvz[:, :conv_dim], qkvz[:, conv_dim:]
        st["ab"] = rnd(N, 2 * hv).to(dt)
        st["conv_state"], st["conv_w"] = rnd(b + 2, CONV - 1, conv_dim).to(dt), (0.5 * rnd(conv_dim, CONV)).to(dt)
        # A in [1, 16] and softplus(dt_bias) in [0.001, 0.1]: the architecture's initial range
        st["ssm_a"] = -torch.exp(torch.rand(hv, device=dev, generator=gen) * math.log(16.0))
        dt_ = torch.exp(torch.rand(hv, device=dev, generator=gen) * math.log(100.0) + math.log(0.001))
        st["dt_bias"] = torch.log(torch.expm1(dt_))
        st["rec"] = 0.1 * rnd(b + 2, hv, dk, dv)
        st["norm_w"] = (1 + 0.1 * rnd(dv)).to(dt)
        return st
    H, G, hd, rd, page = (case[n] for n in ("heads", "kv_heads", "hd", "rd", "page"))
    st["table"], st["plan"], n_pages = _layout(case, dev, gen, page)
    if case["kind"] == "write":
        # one product's rows: [q | gate] of each query head, then k; v of its own
        qk = rnd(N, H * 2 * hd + G * hd).to(dt)
        st["q"], st["k"] = qk[:, :H * 2 * hd].view(N, H, 2 * hd)[..., :hd], qk[:, H * 2 * hd:].view(N, G, hd)
        st["v"] = rnd(N, G, hd).to(dt)
        st["qw"], st["kw"] = (1 + 0.1 * rnd(hd)).to(dt), (1 + 0.1 * rnd(hd)).to(dt)
        st["freq"] = 1.0 / THETA ** (torch.arange(0, rd, 2, dtype=torch.float64, device=dev) / rd)
        st["k_pages"], st["v_pages"] = (rnd(n_pages, G, page, hd).to(dt) for _ in range(2))
        return st
    # keys with a part common to a head's (attention sinks), values of varying size by token
    common = 0.5 * rnd(G, 1, hd)
    st["k_pages"] = torch.empty(n_pages, G, page, hd, dtype=dt, device=dev)
    st["v_pages"] = torch.empty_like(st["k_pages"])
    for i in range(0, n_pages, 1024):  # piece by piece, for memory
        n = min(1024, n_pages - i)
        st["k_pages"][i:i + n] = rnd(n, G, page, hd) + common
        st["v_pages"][i:i + n] = rnd(n, G, page, hd) * torch.exp(0.5 * rnd(n, G, page, 1))
    st["q"] = (rnd(N, G, H // G, hd) + common.view(G, 1, hd)).reshape(N, H, hd).to(dt)
    st["gate"] = rnd(N, H, 2 * hd).to(dt)[..., hd:]
    return st


# ---- one pass ----------------------------------------------------------------------------

def run(state):
    return {"plan": _run_plan, "write": _run_write, "attn": _run_attn, "gdn": _run_gdn}[state["case"]["kind"]](state)


def _run_plan(s):
    P, prompts = s["case"]["page"], s["case"]["prompts"]
    requests, new, lengths, held, table, free, n_free, N = (s[n] for n in ("requests", "new", "lengths", "held", "table", "free",
                                                                           "n_free", "tokens"))
    if own:
        from mlx_gsq_amd.runtime.kernels import paged
        plan = paged.page_plan(requests, new, lengths, held, table, free, n_free, tokens=N, page_size=P)
        kept = table.clone()
        if prompts:
            paged.page_release(requests[:prompts], lengths, held, table, free, n_free)
        return {"cu": plan.cu, "rows": plan.rows, "lens": plan.lens, "pos": plan.pos, "slots": plan.slots, "planned": kept,
                "table": table, "held": held, "lengths": lengths, "free": free, "n_free": n_free}
    dev, B, R, W = new.device, new.shape[0], lengths.shape[0], table.shape[1]
    r, n = requests.long(), new.long()
    inside = (r >= 0) & (r < R)
    at = r.clamp(0, R - 1)
    order = torch.arange(B, device=dev)
    again = ((r[:, None] == r) & (order[:, None] > order)).any(1)
    end = n.clamp(min=0).cumsum(0)
    total = lengths[at].long() + n
    fine = inside & ~again & (n >= 0) & (end <= N) & (total <= W * P)
    need = torch.where(fine, ((total + P - 1) // P - held[at]).clamp(min=0), 0)
    cum = need.cumsum(0)
    served = fine & ((need == 0) | (cum <= n_free))
    need = torch.where(served, need, 0)
    cu = torch.cat([end.new_zeros(1), end]).clamp(max=N)
    # pages: entry i of a sequence's new ones
    col = torch.arange(W, device=dev)
    i = col - held[at].long()[:, None]
    takes = (i >= 0) & (i < need[:, None])
    page = free[(n_free - 1 - (cum - need)[:, None] - i).clamp(0, free.shape[0] - 1)]
    table[at] = torch.where(takes, page, table[at])  # requests of a step are different ones here
    held[at] = held[at] + need.int()
    n_free -= torch.where(served, cum, 0).amax(0, keepdim=True).int()
    lens = torch.where(served, total, 0).int()
    rows = torch.where(served, r, -1).int()
    token = torch.arange(N, device=dev)
    seq = torch.searchsorted(cu[1:].contiguous(), token, right=True).clamp(max=B - 1)
    there = (token < cu[-1]) & served[seq]
    pos = torch.where(there, lengths[at].long()[seq] + token - cu[seq], -1)
    slots = torch.where(there, table[at[seq], (pos // P).clamp(0, W - 1)].long() * P + pos % P, -1)
    kept = table.clone()
    if prompts:  # their pages back, the one taken last first
        r = r[:prompts]
        h = held[r].long()
        first, count = h.cumsum(0) - h, h.sum()
        idx = first[:, None] + col
        back = n_free + count - 1 - idx
        mine = col < h[:, None]
        spare = torch.cat([free, free.new_zeros(1)])  # the last one takes what is not given back
        spare[torch.where(mine, back, free.shape[0])] = table[r]
        free.copy_(spare[:-1])
        table[r] = torch.where(mine, -1, table[r])
        held[r] = 0
        lengths[r] = 0
        n_free += count
    return {"cu": cu.int(), "rows": rows, "lens": lens, "pos": pos, "slots": slots, "planned": kept, "table": table, "held": held,
            "lengths": lengths, "free": free, "n_free": n_free}


def _run_write(s):
    pos, slots = s["plan"][3:]
    if own:
        from mlx_gsq_amd.runtime.kernels import paged
        q = paged.paged_write(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["freq"], s["k_pages"], s["v_pages"], pos, slots,
                              eps=EPS)
        return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}
    c, dt = s["case"], s["q"].dtype
    rd, page = c["rd"], c["page"]
    ang = pos.double()[:, None, None] * s["freq"]
    cos, sin = ang.cos().float(), ang.sin().float()

    def norm_rope(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        lo, hi = x[..., :rd // 2], x[..., rd // 2:rd]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., rd:]], -1).to(dt)
    s["k_pages"][slots // page, :, slots % page] = norm_rope(s["k"], s["kw"])
    s["v_pages"][slots // page, :, slots % page] = s["v"]
    return {"q": norm_rope(s["q"], s["qw"]), "k": s["k_pages"], "v": s["v_pages"]}


def _groups(case):
    """(first sequence, one past the last, most new tokens) of the prompts and of the single tokens."""
    p, b = case["prompts"], case["b"]
    return [g for g in ((0, p, case["new"]), (p, b, 1)) if g[0] < g[1]]


def _run_attn(s):
    c = s["case"]
    if own:
        from mlx_gsq_amd.runtime.kernels import paged
        return paged.attn_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], paged.PagePlan(*s["plan"]), gate=s["gate"],
                                max_new=c["new"])
    H, G, hd, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    cu, rows, lens = s["plan"][:3]
    cached, new = _lengths(c)
    out = torch.empty_like(s["q"])
    for b0, b1, S in _groups(c):
        L = max(x + n for x, n in zip(cached[b0:b1], new[b0:b1]))
        m = b1 - b0
        n = (cu[b0 + 1:b1 + 1] - cu[b0:b1]).long()
        at = (cu[b0:b1].long()[:, None] + torch.arange(S, device=cu.device)).clamp(max=out.shape[0] - 1)   # (m, S)
        table = s["table"][rows[b0:b1].long(), :-(-L // page)].clamp(min=0).long()
        k = s["k_pages"][table].transpose(1, 2).reshape(m, G, -1, hd).float()
        q = s["q"][at].float().view(m, S, G, H // G, hd).permute(0, 2, 3, 1, 4).reshape(m, G, H // G * S, hd)
        scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(m, G, H // G, S, -1) * hd ** -0.5
        del k
        last = (lens[b0:b1] - n)[:, None] + torch.arange(S, device=cu.device)   # (m, S): position of a token
        scores.masked_fill_((torch.arange(scores.shape[-1], device=cu.device) > last[..., None])[:, None, None], float("-inf"))
        p = (scores - scores.amax(-1, keepdim=True)).exp_()
        p = p / p.sum(-1, keepdim=True)
        v = s["v_pages"][table].transpose(1, 2).reshape(m, G, -1, hd).float()
        o = torch.matmul(p.view(m, G, H // G * S, -1), v).view(m, H, S, hd).transpose(1, 2)
        o = (o / (1 + torch.exp(-s["gate"][at].float()))).to(out.dtype)
        lo, hi = sum(new[:b0]), sum(new[:b1])
        seq = torch.repeat_interleave(torch.arange(m, device=cu.device), n, output_size=hi - lo)
        token = torch.arange(lo, hi, device=cu.device)
        out[lo:hi] = o[seq, token - cu[b0:b1].long()[seq]]
    return out


def _run_gdn(s):
    c = s["case"]
    hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
    if own:
        from mlx_gsq_amd.runtime.kernels import paged
        out = paged.gdn_packed(s["qkv"], s["z"], s["ab"], s["conv_state"], s["conv_w"], s["ssm_a"], s["dt_bias"], s["rec"],
                               s["norm_w"], paged.PagePlan(*s["plan"]), key_heads=hk, value_heads=hv, head_k_dim=dk,
                               head_v_dim=dv, eps=EPS, max_new=c["new"])
        return {"out": out, "conv": s["conv_state"], "rec": s["rec"]}
    cu, rows, lens = s["plan"][:3]
    new = _lengths(c)[1]
    out = s["z"].new_empty(s["z"].shape)
    dev = out.device
    for b0, b1, S in _groups(c):
        m, row = b1 - b0, rows[b0:b1].long()
        n = (cu[b0 + 1:b1 + 1] - cu[b0:b1]).long()
        at = (cu[b0:b1].long()[:, None] + torch.arange(S, device=dev)).clamp(max=out.shape[0] - 1)   # (m, S)
        there = torch.arange(S, device=dev) < n[:, None]
        began = (lens[b0:b1] == n).view(m, 1, 1)                             # a request's first tokens: no state yet
        win = torch.cat([torch.where(began, 0, s["conv_state"][row]), s["qkv"][at]], 1)
        keep = n[:, None] + torch.arange(CONV - 1, device=dev)
        s["conv_state"][row] = torch.gather(win, 1, keep[..., None].expand(-1, -1, win.shape[2]))
        acc = sum(win[:, j:j + S].float() * s["conv_w"].float()[:, j] for j in range(CONV))
        x = acc / (1 + torch.exp(-acc))
        q, k, v = x.split([hk * dk, hk * dk, hv * dv], -1)

        def heads(t, size):  # value head h reads the normalized rows of key head h % hk
            t = t.reshape(m, S, hk, dk)
            t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * size
            return t.repeat(1, 1, hv // hk, 1).transpose(1, 2)
        q, k, v = heads(q, 1 / dk), heads(k, dk ** -0.5), v.reshape(m, S, hv, dv).transpose(1, 2)
        a, b = s["ab"][at].float().split(hv, -1)
        beta = (there[..., None] / (1 + torch.exp(-b))).transpose(1, 2)[..., None]        # (m, hv, S, 1)
        a = a.double() + s["dt_bias"]
        g = s["ssm_a"] * torch.where(a > 20, a, torch.log1p(torch.exp(a.clamp(max=20))))
        g = (g * there[..., None]).transpose(1, 2)                                        # (m, hv, S), in 64 bits
        st = torch.where(began[..., None], 0, s["rec"][row])
        outs = []
        for t in range(0, S, CHUNK):
            qc, kc, vc, bc = (y[:, :, t:t + CHUNK] for y in (q, k, v, beta))
            G = g[:, :, t:t + CHUNK].cumsum(-1)
            w = G.shape[-1]
            low = torch.ones(w, w, dtype=torch.bool, device=dev).tril()
            ratio = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, float("-inf"))).float()
            grown, left = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None]
            kt = kc.transpose(2, 3).contiguous()
            mat = bc * ratio * torch.matmul(kc, kt) * low.tril(-1)
            u = bc * (vc - grown * torch.matmul(kc, st))
            for i in range(6):  # (1 + A)^-1 = (1 - A)(1 + A^2)(1 + A^4) ..: 64 tokens
                u = u - torch.matmul(mat, u) if i == 0 else u + torch.matmul(mat, u)
                mat = torch.matmul(mat, mat.contiguous())
            outs.append(grown * torch.matmul(qc, st) + torch.matmul(ratio * torch.matmul(qc, kt), u))
            st = grown[:, :, -1:] * st + torch.matmul(kt, left * u)
        s["rec"][row] = st
        o = torch.cat(outs, 2).transpose(1, 2)                                            # (m, S, hv, dv)
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * s["norm_w"].float()
        z = s["z"][at].float().view(m, S, hv, dv)
        o = (o * z / (1 + torch.exp(-z))).reshape(m, S, hv * dv).to(out.dtype)
        lo, hi = sum(new[:b0]), sum(new[:b1])
        seq = torch.repeat_interleave(torch.arange(m, device=dev), n, output_size=hi - lo)
        out[lo:hi] = o[seq, torch.arange(lo, hi, device=dev) - cu[b0:b1].long()[seq]]
    return {"out": out, "conv": s["conv_state"], "rec": s["rec"]}


# ---- what a pass cannot do without -------------------------------------------------------

def work(case):
    cached, new = _lengths(case)
    N, b = sum(new), case["b"]
    if case["kind"] == "plan":
        total = _pages([c + n for c, n in zip(cached, new)], case["page"])
        taken = sum(total) - sum(_pages(cached, case["page"]))
        # lengths, requests and pages held read, the plan and the pages taken or given back written
        return {"bytes": 16 * N + b * (4 * 4 + 4 * 3) + 8 * taken + 12 * sum(total[:case["prompts"]]), "flops": 8.0 * N}
    if case["kind"] == "gdn":
        hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "dk", "dv"))
        conv_dim = 2 * hk * dk + hv * dv
        rows = 2 * N * (conv_dim + 2 * hv * dv + 2 * hv)
        states = sum((8 if c else 4) * hv * dk * dv + (4 if c else 2) * (CONV - 1) * conv_dim for c in cached)
        return {"bytes": rows + states + 2 * conv_dim * CONV + 2 * dv + 8 * hv + 12 * b,
                "flops": N * (hv * 8.0 * dk * dv + 2.0 * CONV * conv_dim)}
    H, G, hd = case["heads"], case["kv_heads"], case["hd"]
    if case["kind"] == "write":
        return {"bytes": 2 * 2 * N * (H + 2 * G) * hd + 16 * N + 4 * hd + 4 * case["rd"], "flops": 8.0 * N * (H + G) * hd}
    seen = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
    total = sum(c + n for c, n in zip(cached, new))
    return {"bytes": total * G * hd * 4 + N * H * hd * 2 * 3 + 4 * sum(_pages([c + n for c, n in zip(cached, new)], case["page"])),
            "flops": 4.0 * H * hd * seen}


# ---- the definitions in 64 bits ----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return None  # whole numbers
    return {"gdn": _exact_gdn, "write": _exact_write}.get(case["kind"], _exact_attn)(s)


def _exact_write(s):
    c, (pos, slots) = s["case"], s["plan"][3:]
    half, page, hd = c["rd"] // 2, c["page"], c["hd"]
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=pos.device), pos.double()[:, None] * s["freq"])[:, None]

    def turned(x, w):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)
    k, v = s["k_pages"].double(), s["v_pages"].double()
    for cache, x in ((k, turned(s["k"], s["kw"])), (v, s["v"].double())):
        flat = cache.transpose(1, 2).reshape(-1, *x.shape[1:])
        flat[slots] = x
        cache.copy_(flat.view(cache.shape[0], page, -1, hd).transpose(1, 2))
    return {"q": turned(s["q"], s["qw"]), "k": k, "v": v}


def _exact_attn(s):
    c = s["case"]
    H, G, hd, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    cu, rows, lens = (t.tolist() for t in s["plan"][:3])
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, row in enumerate(rows):
        t0, t1, n = cu[b], cu[b + 1], lens[b]
        at = s["table"][row, :-(-n // page)].long()
        later = torch.arange(n, device=out.device) > torch.arange(n - (t1 - t0), n, device=out.device)[:, None]
        for g in range(G):
            k, v = (x[at, g].reshape(-1, hd)[:n].double() for x in (s["k_pages"], s["v_pages"]))
            for h in range(g * (H // G), (g + 1) * (H // G)):
                a = torch.mm(s["q"][t0:t1, h].double(), k.t().contiguous()) / math.sqrt(hd)
                a.masked_fill_(later, -math.inf)
                out[t0:t1, h] = torch.mm((a - torch.logsumexp(a, -1, keepdim=True)).exp(), v)
    return out * torch.sigmoid(s["gate"].double())


def _exact_gdn(s):
    c = s["case"]
    hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
    cu, rows, lens = (t.tolist() for t in s["plan"][:3])
    out = torch.empty(s["z"].shape, dtype=torch.float64, device=s["z"].device)
    conv, rec = s["conv_state"].double(), s["rec"].double()
    head = torch.arange(hv, device=out.device) % hk
    w = s["conv_w"].double()
    for b, row in enumerate(rows):
        t0, t1 = cu[b], cu[b + 1]
        if lens[b] == t1 - t0:
            conv[row], rec[row] = 0, 0
        win = torch.cat([conv[row], s["qkv"][t0:t1].double()])
        conv[row] = win[t1 - t0:]
        x = (win.unfold(0, CONV, 1) * w).sum(-1)
        x = x * torch.sigmoid(x)
        q, k, v = x.split([hk * dk, hk * dk, hv * dv], -1)
        q, k = (y.view(-1, hk, dk) / (y.view(-1, hk, dk).pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() for y in (q, k))
        q, k, v = q[:, head] / dk, k[:, head] / math.sqrt(dk), v.view(-1, hv, dv)
        a, beta = s["ab"][t0:t1].double().split(hv, -1)
        decay = torch.exp(s["ssm_a"].double() * torch.nn.functional.softplus(a + s["dt_bias"].double()))
        beta = torch.sigmoid(beta)
        st, y = rec[row], []
        for t in range(t1 - t0):
            st = st * decay[t, :, None, None]
            st = st + k[t, :, :, None] * (beta[t, :, None] * (v[t] - (st * k[t, :, :, None]).sum(1)))[:, None]
            y.append((st * q[t, :, :, None]).sum(1))
        rec[row] = st
        y = torch.stack(y)
        y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["norm_w"].double()
        z = s["z"][t0:t1].double().view(-1, hv, dv)
        out[t0:t1] = (y * z * torch.sigmoid(z)).view(-1, hv * dv)
    return {"out": out, "conv": conv, "rec": rec}
