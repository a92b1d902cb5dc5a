"""What is timed of the operators for batches that continue one prompt: attention over a shared prefix, the check of drafted tokens,
and the pages of a cache that several sequences hold.

Every case names its operator in ``op``; the classes below hold what a serving program has in hand (``prepare``), one call in its
plain form and through the framework (``plain`` / ``native``), and the call's value in 64 bits (``exact``). Sizes are those of the
configurations in ``triton_distributed_b200/models/config.py`` (head layouts, vocabulary, layers), of the benchmarks and of the tests,
or generic.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _ints(g, low, high, shape, dtype=torch.int32):
    """Whole numbers from low to high, both among them."""
    return torch.randint(low, high + 1, shape, generator=g, device="cuda").to(dtype)


def _log_int(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _pages(tokens, page):
    return -(-tokens // page)


class PrefixAttention:
    """Attention of the last `tokens` tokens of every sequence of a batch whose first `shared` keys are the same pages."""

    @staticmethod
    def prepare(c, seed):
        g = _generator(seed)
        B, T, S, page, H, Hkv, D = (c[n] for n in ("batch", "tokens", "shared", "page", "heads", "kv_heads", "dim"))
        dt = DTYPES[c["dtype"]]
        common, width = S // page, _pages(S + c["own"], page)
        N = common + B * (width - common)
        k, v = (_normal(g, (N, page, Hkv, D), 1.0, dt) for _ in range(2))
        ids = torch.randperm(N, generator=g, device="cuda").to(torch.int32)
        table = torch.empty((B, width), dtype=torch.int32, device="cuda")
        table[:, :common] = ids[:common]
        table[:, common:] = ids[common:].view(B, width - common)
        if S % page:  # the page in which the prompt ends: everybody has a copy of the prompt's last tokens in a page of their own
            first = table[:, common].long()
            for t in (k, v):
                t[first, :S % page] = t[first[0], :S % page].clone()
        lens = S + _ints(g, T, c["own"], (B,))
        lens[0] = S + c["own"]
        live = B - c["padded"]
        lens[live:] = 0       # rows of the batch that hold no sequence
        table[live:] = -1
        # logits of about unit size, as after norms of q and k
        q = _normal(g, (B * T, H, D), 1.0, dt)
        return {"q": q, "k": k, "v": v, "lens": lens, "table": table, "scale": D ** -0.5, "shared": S, "tokens": T, "longest": S + c["own"]}

    @staticmethod
    def native(s):
        from triton_distributed_b200 import ops
        return ops.shared_prefix_attention(s["q"], s["k"], s["v"], s["lens"], s["table"], s["shared"], s["scale"], tokens=s["tokens"],
                                           max_kv_len=s["longest"])

    @staticmethod
    def plain(s):
        q, k, v, lens, table, S, T = s["q"], s["k"], s["v"], s["lens"].long(), s["table"].long(), s["shared"], s["tokens"]
        page, Hkv, D = k.shape[1:]
        B, H = lens.numel(), q.shape[1]
        G = H // Hkv
        k, v = k.view(-1, Hkv, D), v.view(-1, Hkv, D)
        qf = q.view(B, T, Hkv, G, D).float()
        # the shared keys, once for all rows of the batch
        at = torch.arange(S, device=q.device)
        slot = table[0, at // page] * page + at % page
        kp, vp = k[slot].float().transpose(0, 1), v[slot].float().transpose(0, 1)                      # [Hkv, S, D]
        rows = qf.permute(2, 0, 1, 3, 4).reshape(Hkv, B * T * G, D)
        sp = (rows @ kp.transpose(1, 2)).mul_(s["scale"]).view(Hkv, B, T, G, S)
        # everybody's own keys
        pos = torch.arange(S, s["longest"], device=q.device)
        slot = table[:, pos // page].clamp_min(0) * page + pos % page                                  # [B, n]
        ko, vo = k[slot].float(), v[slot].float()                                                      # [B, n, Hkv, D]
        so = (qf.permute(2, 0, 1, 3, 4).reshape(Hkv, B, T * G, D) @ ko.permute(2, 0, 3, 1)).mul_(s["scale"]).view(Hkv, B, T, G, -1)
        limit = lens[:, None] - T + 1 + torch.arange(T, device=q.device)                               # keys that a token sees
        sp.masked_fill_((at >= limit[..., None])[None, :, :, None], -math.inf)
        so.masked_fill_((pos >= limit[..., None])[None, :, :, None], -math.inf)
        top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
        top = torch.where(top == -math.inf, 0.0, top)
        sp, so = sp.sub_(top).exp_(), so.sub_(top).exp_()
        total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
        o = (sp.view(Hkv, B * T * G, S) @ vp).view(Hkv, B, T, G, D) + (so.view(Hkv, B, T * G, -1) @ vo.permute(2, 0, 1, 3)).view(Hkv, B, T, G, D)
        o = torch.where(total > 0, o / total, 0.0)
        return o.permute(1, 2, 0, 3, 4).reshape(B * T, H, D).to(q.dtype)

    @staticmethod
    def exact(c, seed):
        """Sequence by sequence over the pages of its own table."""
        s = PrefixAttention.prepare(c, seed)
        T, H, Hkv, D, page = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["page"]
        out = torch.zeros((c["batch"] * T, H, D), dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            pages = s["table"][b, :_pages(n, page)].long()
            keys, values = (s[x][pages].reshape(-1, Hkv, D)[:n].double() for x in ("k", "v"))
            for t in range(T):
                seen = n - T + t + 1
                x = s["q"][b * T + t].double().view(Hkv, H // Hkv, D)
                w = torch.einsum("kgd,nkd->kgn", x, keys[:seen]) * s["scale"]
                w = torch.exp(w - w.amax(-1, keepdim=True))
                out[b * T + t] = (torch.einsum("kgn,nkd->kgd", w, values[:seen]) / w.sum(-1, keepdim=True)).view(H, D)
        return out

    @staticmethod
    def work(c):
        rows, live = c["batch"] * c["tokens"], c["batch"] - c["padded"]
        mean = (c["own"] + c["tokens"]) / 2
        keys = c["shared"] + live * mean
        return {"bytes": (2 * keys * c["kv_heads"] + 2 * rows * c["heads"]) * c["dim"] * 2,
                "flops": 4 * live * c["tokens"] * c["heads"] * c["dim"] * (c["shared"] + mean)}

    @staticmethod
    def draw(rng):
        heads, kv_heads = rng.choice([(64, 8), (32, 8), (8, 1), (40, 8), (28, 4), (14, 2), (16, 16), (5, 1)])
        c = {"op": "prefix", "batch": _log_int(rng, 1, 256), "tokens": rng.choice([1, 1, 1, 2, 3, 5, 8]), "heads": heads, "kv_heads": kv_heads,
             "dim": rng.choice([64, 128, 128, 128]), "page": rng.choice([16, 32, 48, 64, 64, 128, 256]), "own": _log_int(rng, 8, 1024),
             "dtype": rng.choice(["bf16", "bf16", "f16"]), "padded": 0}
        if c["batch"] > 4:
            c["padded"] = rng.choice([0, 0, 1, c["batch"] // 4])
        rows = c["batch"] * c["tokens"] * heads * c["dim"]
        top = min(131072, (256 * 8 * 128 * 131072) // rows, (1 << 29) // (kv_heads * c["dim"]))
        while c["batch"] * c["own"] * kv_heads * c["dim"] > 1 << 28:
            c["own"] = max(c["tokens"], c["own"] // 2)
        c["shared"] = _log_int(rng, 100, max(101, top))
        return c


class Verify:
    """Which drafted tokens stand, and the token behind them: speculative sampling with the random numbers given."""

    @staticmethod
    def prepare(c, seed):
        g = _generator(seed)
        B, K, V, dt = c["batch"], c["drafts"], c["vocab"], DTYPES[c["dtype"]]
        logits = _normal(g, (B, K + 1, V), 2.5, torch.float32)
        # the draft model's logits are near the target's
        near = logits[:, :K] + _normal(g, (B, K, V), 0.7, torch.float32)
        p = torch.softmax(logits, -1).to(dt)
        q = torch.softmax(near, -1)
        if c["sampled"]:
            gaps = torch.empty_like(q).exponential_(generator=g)
            drafts = (q / gaps).argmax(-1)
        else:            # picked without chance: the draft's best token
            drafts = near.argmax(-1)
            best = torch.rand((B, K), generator=g, device="cuda") < 0.7
            drafts = torch.where(best, logits[:, :K].argmax(-1), drafts)
            p = torch.softmax(logits * 3, -1).to(dt)
        lens = _ints(g, 0, K, (B,)) if c["ragged"] else None
        u = torch.rand((B, K + 1), generator=g, device="cuda")
        return {"drafts": drafts, "p": p, "q": q.to(dt) if c["sampled"] else None, "u": u, "lens": lens}

    @staticmethod
    def native(s):
        from triton_distributed_b200 import ops
        return ops.verify_drafts(s["drafts"], s["p"], s["u"], draft_probs=s["q"], draft_lens=s["lens"])

    @staticmethod
    def plain(s):
        d, p, q, u = s["drafts"], s["p"], s["q"], s["u"].double()
        B, K = d.shape
        V = p.shape[2]
        row, place = torch.arange(B, device=d.device), torch.arange(K, device=d.device)
        lens = s["lens"].long() if s["lens"] is not None else torch.full_like(row, K)
        pd = p[:, :K].gather(2, d[..., None])[..., 0].double()
        qd = q.gather(2, d[..., None])[..., 0].double() if q is not None else torch.ones_like(pd)
        stands = (u[:, :K] * qd < pd) & (place < lens[:, None])
        n = stands.long().cumprod(1).sum(1)
        # the weights of the token behind the accepted ones, in 64 bits: their sums decide between neighbours
        w = p[row, n].double()
        last = n.clamp_max(K - 1)
        if q is not None:
            rest = (w - q[row, last].double()).clamp_min_(0)
        else:
            rest = w.scatter(1, d[row, last][:, None], 0.0)
        rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
        w = torch.where((n < lens)[:, None], rest, w)
        run = w.cumsum(1)
        token = (run <= u[:, K:] * run[:, -1:]).sum(1).clamp_max(V - 1)
        place = torch.arange(K + 1, device=d.device)
        padded = torch.cat([d, d.new_full((B, 1), -1)], 1)
        tokens = torch.where(place < n[:, None], padded, torch.where(place == n[:, None], token[:, None], -1))
        return n.int(), tokens

    @staticmethod
    def exact(c, seed):
        return None  # whole numbers

    @staticmethod
    def work(c):
        row = c["vocab"] * BYTES[c["dtype"]] * (2 if c["sampled"] else 1)
        return {"bytes": c["batch"] * row, "flops": c["batch"] * c["vocab"] * 2}

    @staticmethod
    def draw(rng):
        return {"op": "verify", "batch": _log_int(rng, 1, 256), "drafts": rng.randint(1, 8), "vocab": rng.choice([32003, 50257, 128256, 151936, 151936]),
                "dtype": rng.choice(["f32", "f32", "bf16"]), "sampled": rng.choice([True, True, False]), "ragged": rng.choice([True, False])}


def _pool(c, g, pages):
    """Keys and values of all layers, as a cache keeps them."""
    shape = (c["layers"], pages, c["page"], c["kv_heads"], c["dim"])
    return [_normal(g, shape, 1.0, DTYPES[c["dtype"]]) for _ in range(2)]


class Fork:
    """A prompt's row forked to others, and room for the next tokens of all of them: full pages are shared, the last one is copied."""

    @staticmethod
    def prepare(c, seed):
        g = _generator(seed)
        page, rows = c["page"], c["prompts"] * (1 + c["children"])
        held, width = _pages(c["prompt"], page), _pages(c["prompt"] + 64, page) + 1
        N = c["prompts"] * held + rows * 3 + 8
        ids = torch.randperm(N, generator=g, device="cuda").to(torch.int32)
        table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        refs = torch.zeros(N, dtype=torch.int32, device="cuda")
        lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        table[:c["prompts"], :held] = ids[:c["prompts"] * held].view(c["prompts"], held)
        refs[ids[:c["prompts"] * held].long()] = 1
        lens[:c["prompts"]] = c["prompt"] - _ints(g, 0, min(page, c["prompt"]) // 4, (c["prompts"],))
        table[:c["prompts"]].masked_fill_(torch.arange(width, device="cuda") >= (lens[:c["prompts"], None] + page - 1) // page, -1)
        refs.zero_().index_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
        src = torch.arange(c["prompts"], dtype=torch.int32, device="cuda").repeat_interleave(c["children"])
        dst = torch.arange(c["prompts"], rows, dtype=torch.int32, device="cuda")
        return {"caches": _pool(c, g, N), "table": table, "lens": lens, "refs": refs, "src": src, "dst": dst, "page": page, "count": c["count"]}

    @staticmethod
    def native(s):
        from triton_distributed_b200 import ops
        ops.fork_pages(s["table"], s["lens"], s["refs"], s["src"], s["dst"], s["page"])
        ops.reserve_pages(s["table"], s["lens"], s["refs"], s["count"], s["caches"], dim=1)
        return [s["table"], s["lens"], s["refs"], *s["caches"]]

    @staticmethod
    def plain(s):
        table, lens, refs, src, dst, page, count = (s[n] for n in ("table", "lens", "refs", "src", "dst", "page", "count"))
        R, W = table.shape
        N = refs.numel()
        at = torch.arange(W, device=table.device)
        one = lambda t: torch.ones_like(t, dtype=torch.int32)  # noqa: E731
        # fork: the rows let go of what they held and take the sources' pages
        src, dst = src.long(), dst.long()
        old, new = table[dst], table[src].masked_fill(at >= (lens[src, None] + page - 1) // page, -1)
        refs.index_add_(0, old.clamp_min(0).flatten().long(), -(old >= 0).int().flatten())
        refs.index_add_(0, new.clamp_min(0).flatten().long(), (new >= 0).int().flatten())
        table[dst], lens[dst] = new, lens[src]
        # room: who writes into a page that others hold gets a copy (where all its holders write, the first row keeps it)
        row = torch.arange(R, device=table.device)
        held, need = (table >= 0).sum(1), (lens.long() + count + page - 1) // page
        last, inside = lens.long() // page, lens.long() % page
        part = table[row, last].clamp_min(0).long()
        writes = (inside > 0) & (refs[part] > 1)
        asks = torch.zeros_like(refs).index_add_(0, part, writes.int())
        first = torch.full_like(refs, R).scatter_reduce_(0, part, torch.where(writes, row, R).int(), "amin")
        copy = writes & ~((asks[part] == refs[part]) & (first[part] == row))
        wants = copy + (need - held).clamp_min(0)
        begin = wants.cumsum(0) - wants
        free = torch.sort((refs > 0).int(), stable=True).indices
        fresh = (at >= held[:, None]) & (at < need[:, None])
        given = free[(begin[:, None] + copy[:, None] + at - held[:, None]).clamp(0, N - 1)]
        table.copy_(torch.where(fresh, given, table).int())
        rows = copy.nonzero()[:, 0]
        to = free[begin[rows]]
        table[rows, last[rows]] = to.int()
        refs.index_add_(0, part[rows], -one(rows))
        refs.index_add_(0, to, one(to))
        refs.index_add_(0, given.flatten(), fresh.int().flatten())
        tokens = torch.arange(page, device=table.device) < inside[rows, None]
        for t in s["caches"]:
            t[:, to] = torch.where(tokens[None, :, :, None, None], t[:, part[rows]], t[:, to])
        return [table, lens, refs, *s["caches"]]

    @staticmethod
    def exact(c, seed):
        return None  # nothing is computed: pages move as they are

    @staticmethod
    def work(c):
        inside = max(1, (c["prompt"] - min(c["page"], c["prompt"]) // 8) % c["page"])
        moved = c["prompts"] * c["children"] * inside * c["kv_heads"] * c["dim"] * BYTES[c["dtype"]] * 2 * c["layers"]
        rows = c["prompts"] * (1 + c["children"])
        return {"bytes": 2 * moved + 2 * 4 * rows * _pages(c["prompt"] + 64, c["page"]), "flops": 0}

    @staticmethod
    def draw(rng):
        c = {"op": "fork", "prompts": rng.choice([1, 1, 2, 5]), "children": _log_int(rng, 1, 32), "prompt": _log_int(rng, 20, 4000), "count": rng.choice([1, 1, 5, 9]),
             "layers": _log_int(rng, 2, 64), "kv_heads": rng.choice([1, 2, 8]), "dim": rng.choice([64, 128]), "page": rng.choice([16, 48, 64, 128]),
             "dtype": rng.choice(["bf16", "f16", "f32"])}
        pages = c["prompts"] * (_pages(c["prompt"], c["page"]) + (1 + c["children"]) * 3) + 8
        size = pages * c["page"] * c["kv_heads"] * c["dim"] * BYTES[c["dtype"]] * 2
        c["layers"] = max(1, min(c["layers"], (3 << 30) // size))
        return c


class Compact:
    """The pages in use moved to the front of a cache that has been used for a while."""

    @staticmethod
    def prepare(c, seed):
        g = _generator(seed)
        N, R, W = c["pages"], c["rows"], c["width"]
        ids = torch.randperm(N, generator=g, device="cuda").to(torch.int32)
        held = _ints(g, 1, W, (R,))
        at = torch.arange(W, device="cuda")
        common = W // 4       # what the rows of a pair have in common
        mine = ids[torch.arange(R * W, device="cuda") % int(N * c["used"])].view(R, W)
        mine[:, :common] = mine[torch.arange(R, device="cuda") // 2 * 2, :common]
        table = torch.where(at < held[:, None], mine, -1).int()
        refs = torch.zeros(N, dtype=torch.int32, device="cuda")
        there = table[table >= 0].long()
        refs.index_add_(0, there, torch.ones_like(there, dtype=torch.int32))
        return {"caches": _pool(c, g, N), "table": table, "refs": refs}

    @staticmethod
    def native(s):
        from triton_distributed_b200 import ops
        table, refs = ops.compact_pages(s["table"], s["refs"], s["caches"], dim=1)
        return [table, refs, *s["caches"]]

    @staticmethod
    def plain(s):
        table, refs = s["table"], s["refs"]
        ids, live = torch.arange(refs.numel(), device=refs.device), refs > 0
        front = ids < live.sum()
        src, dst = (live & ~front).nonzero()[:, 0], (~live & front).nonzero()[:, 0]
        for t in s["caches"]:
            t[:, dst] = t[:, src]
        to = ids.int()
        to[src] = dst.int()
        moved = refs.clone()
        moved[dst], moved[src] = refs[src], 0
        return [torch.where(table >= 0, to[table.clamp_min(0).long()], -1), moved, *s["caches"]]

    @staticmethod
    def exact(c, seed):
        return None  # nothing is computed: pages move as they are

    @staticmethod
    def work(c):
        live = min(c["pages"] * c["used"], c["rows"] * c["width"]) * 0.55      # rows hold half of their width, and share some of it
        moved = live * (1 - live / c["pages"])
        page = c["page"] * c["kv_heads"] * c["dim"] * BYTES[c["dtype"]] * 2 * c["layers"]
        return {"bytes": 2 * moved * page + 4 * (2 * c["rows"] * c["width"] + 2 * c["pages"]), "flops": 0}

    @staticmethod
    def draw(rng):
        c = {"op": "compact", "pages": _log_int(rng, 40, 2048), "rows": _log_int(rng, 2, 200), "used": rng.choice([0.3, 0.6, 0.9]), "layers": _log_int(rng, 1, 32),
             "kv_heads": rng.choice([1, 2, 8]), "dim": rng.choice([64, 128]), "page": rng.choice([16, 48, 64]), "dtype": rng.choice(["bf16", "f16", "f32"])}
        c["width"] = max(4, int(c["pages"] * c["used"]) // c["rows"])
        size = c["pages"] * c["page"] * c["kv_heads"] * c["dim"] * BYTES[c["dtype"]] * 2
        c["layers"] = max(1, min(c["layers"], (3 << 30) // size))
        return c


OPERATORS = {"prefix": PrefixAttention, "verify": Verify, "fork": Fork, "compact": Compact}


def listed():
    attention = {"op": "prefix", "tokens": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "padded": 0}
    return [
        # two samples of a short prompt: what a call costs at the least
        {**attention, "name": "prefix two samples", "batch": 2, "heads": 32, "shared": 1000, "own": 64},
        # sixteen samples of the benchmark's prompt length
        {**attention, "name": "prefix sixteen samples", "batch": 16, "shared": 2048, "own": 512},
        # drafted tokens being verified: five query tokens a sequence, small pages, an odd prompt length, a batch that is not full
        {**attention, "name": "prefix drafts", "batch": 24, "tokens": 5, "heads": 40, "page": 16, "shared": 7001, "own": 300, "dtype": "f16", "padded": 2},
        # narrow heads
        {**attention, "name": "prefix narrow heads", "batch": 48, "tokens": 3, "heads": 14, "kv_heads": 2, "dim": 64, "page": 32, "shared": 16384, "own": 700},
        # a long document, many questions
        {**attention, "name": "prefix long", "batch": 64, "shared": 32768, "own": 1024},
        # one rank's heads of an 8-way split, a very long document, the largest batch
        {**attention, "name": "prefix shard", "batch": 256, "heads": 8, "kv_heads": 1, "page": 128, "shared": 131072, "own": 256},
        # one sequence, four drafts
        {"op": "verify", "name": "verify one", "batch": 1, "drafts": 4, "vocab": 151936, "dtype": "f32", "sampled": True, "ragged": False},
        # a serving batch
        {"op": "verify", "name": "verify batch", "batch": 64, "drafts": 5, "vocab": 151936, "dtype": "f32", "sampled": True, "ragged": False},
        # drafts looked up in the text itself (no probabilities), of different lengths, a vocabulary of odd size, 16-bit probabilities
        {"op": "verify", "name": "verify lookup", "batch": 200, "drafts": 8, "vocab": 32003, "dtype": "bf16", "sampled": False, "ragged": True},
        # four samples of a short prompt in a small model
        {"op": "fork", "name": "fork few", "prompts": 1, "children": 3, "prompt": 100, "count": 1, "layers": 4, "kv_heads": 2, "dim": 128, "page": 64, "dtype": "bf16"},
        # sixteen samples of two prompts, 64 layers
        {"op": "fork", "name": "fork many", "prompts": 2, "children": 15, "prompt": 1000, "count": 5, "layers": 64, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # a cache of which half is in use, in no order
        {"op": "compact", "name": "compact", "pages": 512, "rows": 32, "width": 15, "used": 0.95, "layers": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
    ]


def draw(rng):
    return OPERATORS[rng.choice(["prefix", "prefix", "prefix", "verify", "verify", "fork", "compact"])].draw(rng)


def prepare(case, seed):
    return {"op": case["op"], **OPERATORS[case["op"]].prepare(case, seed)}


def run(state):
    operator = OPERATORS[state["op"]]
    if own:
        return operator.native(state)
    return operator.plain(state)


def work(case):
    return OPERATORS[case["op"]].work(case)


def exact(case, seed):
    return OPERATORS[case["op"]].exact(case, seed)
