"""Plain references of the operators over packed sequences and paged caches: whole numbers on lists, the rest in float64
on the CPU, sequence by sequence from the definitions."""
import math

import torch

F16, BF16 = torch.float16, torch.bfloat16


def gen(*key):
    seed = 0
    for x in key:
        for ch in str(x):
            seed = (seed * 131 + ord(ch)) % (1 << 31)
    return torch.Generator().manual_seed(seed)


# ---- plans ---------------------------------------------------------------------------------------

def plan(requests, new, lengths, held, table, free, n_free, tokens, page):
    """The step of ``page_plan`` on lists (table: rows of lists); changes held and table, returns the plan and n_free."""
    B, R, W = len(requests), len(lengths), len(table[0])
    ends, taken, cum, rows, lens = [], 0, 0, [], []
    stop = 0
    start_held = list(held)
    for b in range(B):
        r, n = requests[b], new[b]
        stop += max(n, 0)
        ends.append(min(stop, tokens))
        fine = 0 <= r < R and r not in requests[:b] and n >= 0 and stop <= tokens
        fine = fine and lengths[r] >= 0 and 0 <= start_held[r] <= W and lengths[r] + n <= W * page
        if fine:
            need = max(0, -(-(lengths[r] + n) // page) - start_held[r])
            cum += need
            fine = need == 0 or cum <= n_free
        if not fine:
            rows.append(-1)
            lens.append(0)
            continue
        for i in range(need):
            table[r][start_held[r] + i] = free[n_free - 1 - (cum - need) - i]
        held[r] += need
        taken += need
        rows.append(r)
        lens.append(lengths[r] + n)
    cu = [0] + ends
    pos, slots = [-1] * tokens, [-1] * tokens
    for b in range(B):
        if rows[b] >= 0:
            for i in range(cu[b + 1] - cu[b]):
                p = lens[b] - (cu[b + 1] - cu[b]) + i
                pos[cu[b] + i] = p
                slots[cu[b] + i] = table[rows[b]][p // page] * page + p % page
    return (cu, rows, lens, pos, slots), n_free - taken


def release(requests, lengths, held, table, free, n_free):
    out = []
    for b, r in enumerate(requests):
        if 0 <= r < len(lengths) and r not in requests[:b]:
            out += table[r][:held[r]]
            table[r][:held[r]] = [-1] * held[r]
            held[r] = lengths[r] = 0
    for p in reversed(out):
        free[n_free] = p
        n_free += 1
    return n_free


def step(cached, new, page, g, spare_requests=2, spare_pages=2, tail=0):
    """A step over pages in random order: (table, plan as tensors, number of pages). tail: rows behind the last sequence."""
    total = [c + n for c, n in zip(cached, new)]
    need = [-(-t // page) for t in total]
    B, R = len(new), len(new) + spare_requests
    n_pages = sum(need) + spare_pages
    order = torch.randperm(n_pages, generator=g).tolist()
    rows = torch.randperm(R, generator=g).tolist()[:B]
    W = max(need + [1]) + 1
    table = [[-1] * W for _ in range(R)]
    for b in range(B):
        table[rows[b]][:need[b]] = [order.pop() for _ in range(need[b])]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    pos, slots = [], []
    for b in range(B):
        for p in range(cached[b], total[b]):
            pos.append(p)
            slots.append(table[rows[b]][p // page] * page + p % page)
    pos += [-1] * tail
    slots += [-1] * tail
    i32, i64 = torch.int32, torch.int64
    return (torch.tensor(table, dtype=i32), (torch.tensor(cu, dtype=i32), torch.tensor(rows, dtype=i32),
                                             torch.tensor(total, dtype=i32), torch.tensor(pos, dtype=i64),
                                             torch.tensor(slots, dtype=i64)), n_pages)


# ---- attention -----------------------------------------------------------------------------------

def attention(q, k_pages, v_pages, table, cu, rows, lens, gate=None):
    """(out, sum of weights times |V| times the gate, largest sum |q k| / sqrt(hd) of a row), float64, for served sequences;
    zeros elsewhere."""
    N, H, hd = q.shape
    G, P = k_pages.shape[1:3]
    out, size, score = (torch.zeros(N, H, hd, dtype=torch.float64) for _ in range(3))
    for b in range(len(rows)):
        t0, t1, n, r = int(cu[b]), int(cu[b + 1]), int(lens[b]), int(rows[b])
        if r < 0 or t1 <= t0:
            continue
        at = table[r, :-(-n // P)].long()
        last = torch.arange(n - (t1 - t0), n)
        later = torch.arange(n) > last[:, None]
        for h in range(H):
            g = h // (H // G)
            k, v = (x[at, g].reshape(-1, hd)[:n].double() for x in (k_pages, v_pages))
            qh = q[t0:t1, h].double()
            s = (qh @ k.T) / math.sqrt(hd)
            s[later] = -math.inf
            p = torch.softmax(s, -1)
            finite = torch.isfinite(v).all(-1)
            if bool(finite.all()):
                o = p @ v
            else:  # what a token does not see does not reach it: 0 times anything
                o = torch.stack([p[i, :int(last[i]) + 1] @ v[:int(last[i]) + 1] for i in range(t1 - t0)])
            out[t0:t1, h], size[t0:t1, h] = o, p @ v.abs().nan_to_num(0, 0, 0)
            score[t0:t1, h] = ((qh.abs() @ k.abs().T) / math.sqrt(hd)).masked_fill(later, 0).amax(-1, keepdim=True).expand(-1, hd)
    if gate is not None:
        out, size = out * torch.sigmoid(gate.double()), size * torch.sigmoid(gate.double())
    return out, size, score


def attention_bound(want, size, score, dtype, hd, L):
    """What the kernels' roundings allow: one of the output to dtype; scores of hd products, matrix cores that truncate
    up to 4 times for 32 products (2^-23 each, of the sum of the products' sizes), which move a weight by twice that; sums over L
    positions alike; weights held in 22 (fp16) or 16 (bf16) bits; a few ulps of float32 for exp, the division and the gate."""
    eps = torch.finfo(dtype).eps / 2
    rel = 2 * (hd / 8 + 2) * 2.0 ** -23 * score + (L / 8 + 16) * 2.0 ** -23 + (2.0 ** -22 if dtype is F16 else 2.0 ** -16)
    return eps * want.abs() + rel * size * (1 + eps) + 2.0 ** -25


# ---- GatedDeltaNet -------------------------------------------------------------------------------

def gdn(qkv, z, ab, conv, conv_w, ssm_a, dt_bias, rec, norm_w, cu, rows, lens, hk, hv, dk, dv, eps):
    """(out, conv states, rec states, |norm_w silu(z)|) in float64; rows of sequences that are not served stay zeros."""
    N, K = qkv.shape[0], conv_w.shape[-1]
    out = torch.zeros(N, hv * dv, dtype=torch.float64)
    conv, rec = conv.double().clone(), rec.double().clone()
    head = torch.arange(hv) % hk
    for b in range(len(rows)):
        t0, t1, r = int(cu[b]), int(cu[b + 1]), int(rows[b])
        if r < 0 or t1 <= t0:
            continue
        if int(lens[b]) == t1 - t0:
            conv[r], rec[r] = 0, 0
        win = torch.cat([conv[r], qkv[t0:t1].double()])
        conv[r] = win[t1 - t0:]
        x = (win.unfold(0, K, 1) * conv_w.double()).sum(-1)
        x = x * torch.sigmoid(x)
        q, k, v = x.split([hk * dk, hk * dk, hv * dv], -1)
        q, k = (y.view(-1, hk, dk) / (y.view(-1, hk, dk).pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() for y in (q, k))
        q, k, v = q[:, head] / dk, k[:, head] / math.sqrt(dk), v.view(-1, hv, dv)
        a, beta = ab[t0:t1].double().split(hv, -1)
        decay = torch.exp(ssm_a.double() * torch.nn.functional.softplus(a + dt_bias.double()))
        beta = torch.sigmoid(beta)
        st, ys = rec[r].clone(), []
        for t in range(t1 - t0):
            st = st * decay[t, :, None, None]
            st = st + k[t, :, :, None] * (beta[t, :, None] * (v[t] - (st * k[t, :, :, None]).sum(1)))[:, None]
            ys.append((st * q[t, :, :, None]).sum(1))
        rec[r] = st
        y = torch.stack(ys)
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * norm_w.double()
        zz = z[t0:t1].double().view(-1, hv, dv)
        out[t0:t1] = (y * zz * torch.sigmoid(zz)).reshape(t1 - t0, -1)
    zz = z.double().view(N, hv, dv)
    return out, conv, rec, (norm_w.double() * zz * torch.sigmoid(zz)).abs().view(N, -1)
