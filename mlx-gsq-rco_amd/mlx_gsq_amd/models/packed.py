"""Serving many requests with the Qwen3.5-hybrid decoder: their states in one ``PagedCache``, the new tokens of a step
packed behind one another (``Qwen35Model.step``), single-token steps captured in a graph (``PackedGraphDecoder``).

The reference serves one sequence at a time (mlx-lm's generation over mlx_gsq/models/qwen35.py:114-152). On a GPU a
step runs the kernels of runtime/kernels/paged.py; the formulations here and in qwen35.py compute the same for CPU tensors.
"""
from __future__ import annotations

import torch


def _numbers(requests):
    """Requests as int32; what does not fit is out of range there too."""
    t = torch.as_tensor(requests)
    if t.is_floating_point() and t.numel():
        raise ValueError("requests are whole numbers")
    return t.to(torch.int64).clamp(-1, 2 ** 31 - 1).to(torch.int32)


class PagedCache:
    """States of up to ``requests`` requests. K and V of the attention layers lie in ``pages`` pages of ``page_size`` positions,
    handed out as requests grow (up to ``max_len`` positions each, which is rounded up to whole pages); the GatedDeltaNet
    layers keep a state for each request.

    All bookkeeping is on the device: ``table`` (requests, max_pages), ``lengths`` and ``held`` (requests,), ``free`` and
    ``n_free``, int32. A request begins with its first tokens at length 0 and ends with ``release``.

    A step that fails part way has advanced the recurrent states of some layers and no lengths: run again, it would
    advance them twice. ``torn`` then holds the requests that it served and that are not released yet, and no step is taken
    until there are none.
    """

    def __init__(self, args, requests: int, pages: int, page_size: int, max_len: int, device, dtype):
        from ..runtime.kernels.paged import PAGE_SIZES
        device = torch.device(device)
        if page_size not in PAGE_SIZES:
            raise ValueError(f"a page holds one of {PAGE_SIZES} positions, not {page_size}")
        if requests < 1 or pages < 1 or max_len < 1:
            raise ValueError("a cache holds at least one request, page and position")
        if device.type == "cuda":
            if dtype not in (torch.float16, torch.bfloat16):
                raise ValueError(f"paged caches hold 16-bit values, not {dtype}")
            if (args.head_dim not in (64, 128, 256) or args.linear_key_head_dim not in (32, 64, 128)
                    or args.linear_value_head_dim not in (64, 128, 256)):
                raise ValueError("head dims must be 64, 128 or 256 (GatedDeltaNet keys 32, 64 or 128)")
        max_len = -(-max_len // page_size) * page_size
        self.args, self.requests, self.page_size, self.max_len = args, requests, page_size, max_len
        i32 = dict(dtype=torch.int32, device=device)
        self.table = torch.full((requests, max_len // page_size), -1, **i32)
        self.lengths, self.held = torch.zeros(requests, **i32), torch.zeros(requests, **i32)
        self.free, self.n_free = torch.arange(pages, **i32), torch.tensor([pages], **i32)
        self.torn = None
        self.conv, self.rec, self.k, self.v = {}, {}, {}, {}
        for i in range(args.num_hidden_layers):
            if args.is_linear(i):
                self.conv[i] = torch.zeros(requests, args.linear_conv_kernel_dim - 1, args.conv_dim, device=device, dtype=dtype)
                self.rec[i] = torch.zeros(requests, args.linear_num_value_heads, args.linear_key_head_dim,
                                          args.linear_value_head_dim, device=device, dtype=torch.float32)
            else:
                shape = (pages, args.num_key_value_heads, page_size, args.head_dim)
                self.k[i], self.v[i] = (torch.zeros(shape, device=device, dtype=dtype) for _ in range(2))

    def whole(self):
        """Refuses a cache that a failed step has left torn."""
        if self.torn is not None and not bool((self.torn >= 0).any()):
            self.torn = None  # it served nobody
        if self.torn is not None:
            raise ValueError("a step over this cache failed part way: release its requests (torn) before the next one")

    def plan(self, requests, new, tokens: int):
        """The layout of a step (``page_plan``) over ``tokens`` rows; takes the pages it needs."""
        if self.table.is_cuda:
            from ..runtime.kernels import paged
            return paged.page_plan(requests, new, self.lengths, self.held, self.table, self.free, self.n_free, tokens=tokens,
                                   page_size=self.page_size)
        return _plan_host(self, requests.tolist(), new.tolist(), tokens)

    def advance(self, plan):
        """The step's tokens are cached."""
        if self.table.is_cuda:
            from ..runtime.kernels import paged
            paged.page_advance(plan, self.lengths)
        else:
            served = plan.rows >= 0
            self.lengths[plan.rows[served].long()] = plan.lens[served]

    def release(self, requests):
        """Ends requests: their pages are free again. Numbers out of range, or named before, are passed over."""
        requests = _numbers(requests).reshape(-1).to(self.table.device)
        if self.table.is_cuda:
            from ..runtime.kernels import paged
            for some in requests.split(paged.MAX_SEQUENCES):
                paged.page_release(some.contiguous(), self.lengths, self.held, self.table, self.free, self.n_free)
        else:
            self._release_host(requests)
        if self.torn is not None:
            gone = set(requests.tolist())
            left = [r for r in self.torn.tolist() if 0 <= r < self.requests and r not in gone]
            self.torn = torch.tensor(left, dtype=torch.int32) if left else None

    def _release_host(self, requests):
        """``page_release`` for a cache on the CPU."""
        back = []
        for r in dict.fromkeys(requests.tolist()):
            if 0 <= r < self.requests:
                n = int(self.held[r])
                back += self.table[r, :n].tolist()
                self.table[r, :n] = -1
                self.held[r] = self.lengths[r] = 0
        n = int(self.n_free)
        self.free[n:n + len(back)] = torch.tensor(back[::-1], dtype=torch.int32)
        self.n_free += len(back)


def _plan_host(c: PagedCache, requests, new, tokens: int):
    """``page_plan`` for a cache on the CPU."""
    from ..runtime.kernels.paged import PagePlan
    P, W, n_free = c.page_size, c.table.shape[1], int(c.n_free)
    held, lengths = c.held.tolist(), c.lengths.tolist()
    cu, rows, lens = [0], [], []
    pos, slots = torch.full((2, tokens), -1, dtype=torch.int64)
    total = taken = asked = 0
    for b, (r, n) in enumerate(zip(requests, new)):
        start, total = total, total + max(n, 0)
        cu.append(min(total, tokens))
        fine = 0 <= r < c.requests and r not in requests[:b] and n >= 0 and total <= tokens and lengths[r] + n <= W * P
        need = max(0, -(-(lengths[r] + n) // P) - held[r]) if fine else 0
        asked += need
        if not fine or (need and asked > n_free):
            rows.append(-1)
            lens.append(0)
            continue
        if need:
            c.table[r, held[r]:held[r] + need] = c.free[n_free - asked:n_free - asked + need].flip(0)
            c.held[r] += need
            taken = asked
        rows.append(r)
        lens.append(lengths[r] + n)
        at = torch.arange(lengths[r], lengths[r] + n)
        pos[start:total] = at
        slots[start:total] = c.table[r].long()[at // P] * P + at % P
    c.n_free -= taken
    i32 = torch.int32
    return PagePlan(torch.tensor(cu, dtype=i32), torch.tensor(rows, dtype=i32), torch.tensor(lens, dtype=i32), pos, slots)


class PackedStep:
    """What the layers of one step share: the cache, the step's plan, and the most new tokens of a sequence."""

    def __init__(self, cache: PagedCache, plan, max_new: int):
        self.cache, self.plan, self.max_new = cache, plan, max_new

    def sequences(self):
        """(request, first row, one past the last, length) of the sequences served, on the host."""
        cu, rows, lens = (t.tolist() for t in self.plan[:3])
        return [(r, cu[b], cu[b + 1], lens[b]) for b, r in enumerate(rows) if r >= 0 and cu[b + 1] > cu[b]]


class PackedGraphDecoder:
    """Steps of one token for each of up to ``batch`` requests of ``cache``, captured once in a HIP graph and replayed: a
    replay plans its step on the device, so requests may join, grow and end between steps.

    ``step(ids, requests)`` returns the logits buffer, rows of the sequences in turn, overwritten by the next step; rows of
    sequences that were not served (no pages left, a full table row) are NaN, and ``plan.rows`` is -1 there.
    """

    def __init__(self, model, cache: PagedCache, batch: int):
        self.model, self.cache, self.batch = model, cache, batch
        device = cache.table.device
        self.ids = torch.zeros(batch, dtype=torch.int64, device=device)
        self.requests = torch.full((batch,), -1, dtype=torch.int32, device=device)
        self.new = torch.zeros(batch, dtype=torch.int32, device=device)
        # one eager step first, of no sequences, which changes nothing: libraries allocate their tables and
        # workspaces outside the capture
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            self._run()
            torch.cuda.synchronize(device)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=side):
                self.logits, self.plan = self._run()
        torch.cuda.current_stream(device).wait_stream(side)
        torch.cuda.synchronize(device)
        self.capture_stream = side  # the graph's QMM launches use its workspace

    def _run(self):
        plan = self.cache.plan(self.requests, self.new, self.batch)
        return self.model._packed(self.ids, plan, self.cache, 1, False), plan

    def step(self, ids, requests):
        n = len(requests)
        if len(ids) != n or n > self.batch:
            raise ValueError(f"one token for each of at most {self.batch} requests")
        self.cache.whole()
        self.ids[:n].copy_(torch.as_tensor(ids, dtype=torch.int64))
        self.requests.fill_(-1)
        self.requests[:n].copy_(_numbers(requests))
        self.new.zero_()
        self.new[:n].fill_(1)
        self.graph.replay()
        return self.logits[:n]
