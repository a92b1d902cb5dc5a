"""Reference semantics of the operators for several continuations of one prompt: attention over a shared prefix, the check of drafted
tokens, and the pages that several sequences hold."""
from __future__ import annotations

import torch


def shared_prefix_attention_ref(q, k_cache, v_cache, kv_lens, block_table, shared: int, scale: float, tokens: int = 1, prefix_table=None):
    """Arguments as ``ops.shared_prefix_attention``; in fp64, sequence by sequence. Returns (out [B * tokens, Hq, D], lse [B * tokens, Hq])."""
    T, Hq, D = q.shape
    num_blocks, page, Hkv, _ = k_cache.shape
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((T, Hq), float("-inf"), dtype=torch.float64, device=q.device)
    common = block_table[0] if prefix_table is None and shared else prefix_table
    for b in range(kv_lens.numel()):
        n = max(0, int(kv_lens[b]))
        at = torch.arange(n, device=q.device)
        pages = block_table[b].long()
        blk = pages[at // page] if n else at
        if shared and n - tokens + 1 >= shared:
            first = at < shared
            blk = torch.where(first, common.long()[(at // page).clamp_max(common.numel() - 1)], blk)
        valid = (blk >= 0) & (blk < num_blocks)
        slot = torch.where(valid, blk, 0) * page + at % page
        k = torch.where(valid[:, None, None], k_cache.view(-1, Hkv, D)[slot].double(), 0.0)
        v = torch.where(valid[:, None, None], v_cache.view(-1, Hkv, D)[slot].double(), 0.0)
        for t in range(tokens):
            seen = n - tokens + t + 1
            if seen <= 0:
                continue
            row = b * tokens + t
            s = torch.einsum("kgd,nkd->kgn", q[row].double().view(Hkv, Hq // Hkv, D), k[:seen]) * scale
            lse[row] = torch.logsumexp(s, -1).view(Hq)
            out[row] = torch.einsum("kgn,nkd->kgd", torch.softmax(s, -1), v[:seen]).reshape(Hq, D)
    return out, lse


def verify_drafts_ref(drafts, target_probs, uniform, draft_probs=None, draft_lens=None):
    """Arguments and results as ``ops.verify_drafts``; in fp64, sequence by sequence."""
    B, K = drafts.shape
    V = target_probs.shape[2]
    clean = lambda x: torch.where((x > 0) & torch.isfinite(x), x, torch.zeros_like(x)).double()  # noqa: E731
    accepted = torch.zeros(B, dtype=torch.int32)
    tokens = torch.full((B, K + 1), -1, dtype=torch.int64)
    for b in range(B):
        n_drafts = K if draft_lens is None else min(K, max(0, int(draft_lens[b])))
        u = uniform[b].double()
        n = 0
        while n < n_drafts:
            d = int(drafts[b, n])
            if not 0 <= d < V:
                break
            q = 1.0 if draft_probs is None else float(clean(draft_probs[b, n, d]))
            if not float(u[n]) * q < float(clean(target_probs[b, n, d])):
                break
            tokens[b, n] = d
            n += 1
        w = clean(target_probs[b, n])
        if n < n_drafts:
            rest = w.clone()
            if draft_probs is not None:
                rest = (w - clean(draft_probs[b, n])).clamp_min(0)
            elif 0 <= int(drafts[b, n]) < V:
                rest[int(drafts[b, n])] = 0
            w = rest if float(rest.sum()) > 0 else w
        run = w.cumsum(0)
        above = (run > max(float(u[K]) * float(run[-1]), 0.0)).nonzero()
        some = (w > 0).nonzero()
        tokens[b, n] = int(above[0]) if len(above) else int(some[-1]) if len(some) else -1
        accepted[b] = n
    return accepted.to(drafts.device), tokens.to(drafts.device)


def fork_pages_ref(block_table, kv_lens, refs, src, dst, page_size: int):
    """New (block_table, kv_lens, refs) as ``ops.fork_pages`` leaves them."""
    table, lens, refs = block_table.clone(), kv_lens.clone(), refs.clone()
    R, N, seen = table.shape[0], refs.numel(), set()
    for s, d in zip(list(map(int, src)), list(map(int, dst))):
        if d in seen or not (0 <= s < R and 0 <= d < R):
            continue
        seen.add(d)
        n = max(0, int(kv_lens[s]))
        row = block_table[s].clone()
        row[-(-n // page_size):] = -1
        for old in block_table[d].tolist():
            if 0 <= old < N:
                refs[old] -= 1
        for new in row.tolist():
            if 0 <= new < N:
                refs[new] += 1
        table[d], lens[d] = row, n
    return table, lens, refs


def trim_pages_ref(block_table, kv_lens, refs, page_size: int, lens=None, rows=None):
    """New (block_table, kv_lens, refs) as ``ops.trim_pages`` leaves them."""
    table, old, refs = block_table.clone(), kv_lens.clone(), refs.clone()
    rows = list(range(table.shape[0])) if rows is None else list(map(int, rows))
    for i, r in enumerate(rows):
        want = 0 if lens is None else int(lens[i])
        if want < 0 or not 0 <= r < table.shape[0]:
            continue
        old[r] = min(int(old[r]), want)
        for w in range(-(-max(0, int(old[r])) // page_size), table.shape[1]):
            if 0 <= int(table[r, w]) < refs.numel():
                refs[int(table[r, w])] -= 1
            table[r, w] = -1
    return table, old, refs


def reserve_pages_ref(block_table, kv_lens, refs, count, page_size: int):
    """(status, new block_table, new refs, copies [(from, to, tokens)]) as ``ops.reserve_pages`` leaves them."""
    table, new = block_table.clone(), refs.clone()
    R, W = table.shape
    counts = [int(c) for c in count] if isinstance(count, torch.Tensor) else [int(count)] * R
    part = {}
    for r in range(R):
        n, c = max(0, int(kv_lens[r])), counts[r]
        if c > 0 and n % page_size and n // page_size < W:
            pg = int(table[r, n // page_size])
            if 0 <= pg < refs.numel() and int(refs[pg]) > 1:
                part.setdefault(pg, []).append(r)
    copies_of = {r: pg for pg, rs in part.items() for r in (rs[1:] if len(rs) == int(refs[pg]) else rs)}
    free = [i for i in range(refs.numel()) if int(refs[i]) <= 0]
    copies, given, gap = [], 0, False

    def take():
        nonlocal given
        given += 1
        return free[given - 1] if given <= len(free) else -1

    for r in range(R):
        n, c = max(0, int(kv_lens[r])), counts[r]
        if c <= 0:
            continue
        need = -(-(n + c) // page_size)
        if need > W:
            return 2, block_table.clone(), refs.clone(), []
        gap = gap or (n > 0 and int(block_table[r, -(-n // page_size) - 1]) < 0)
        held = -(-n // page_size)
        while held < need and int(table[r, held]) >= 0:
            held += 1
        if r in copies_of:
            to = take()
            copies.append((copies_of[r], to, n % page_size))
            table[r, n // page_size] = to
            new[copies_of[r]] -= 1
            new[to] = 1
        for w in range(held, need):
            table[r, w] = take()
            new[table[r, w].long()] = 1
    if gap:
        return 3, block_table.clone(), refs.clone(), []
    if given > len(free):
        return 1, block_table.clone(), refs.clone(), []
    return 0, table, new, copies


def compact_pages_ref(block_table, refs):
    """(new block_table, new refs, moves [(from, to)]) as ``ops.compact_pages`` leaves them."""
    live = [i for i in range(refs.numel()) if int(refs[i]) > 0]
    used = set(live)
    moves = list(zip([i for i in live if i >= len(live)], [i for i in range(len(live)) if i not in used]))
    to = {a: b for a, b in moves}
    table = block_table.clone()
    for i, pg in enumerate(block_table.flatten().tolist()):
        table.view(-1)[i] = to.get(pg, pg)
    new = refs.clone()
    for a, b in moves:
        new[b], new[a] = refs[a], 0
    return table, new, moves
