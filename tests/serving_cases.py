"""Inputs of the tests of shared-prefix attention, draft verification and shared pages: small batches in random states, made on the CPU."""
import torch


def prefix_batch(B, T, Hq, Hkv, D, page, shared, own, dtype=torch.bfloat16, seed=0, lens=None, device="cpu", spare=3):
    """A batch whose rows begin with the same `shared` keys: whole pages are shared, the page in which the shared keys end is everybody's
    copy. Slots that hold no key are NaN. ``lens``: kv_lens (default: shared plus T ... own)."""
    g = torch.Generator().manual_seed(seed)
    width = -(-(shared + own) // page)
    common = shared // page
    N = common + B * (width - common) + spare
    k, v = torch.randn(N, page, Hkv, D, generator=g), torch.randn(N, page, Hkv, D, generator=g)
    ids = torch.randperm(N, generator=g).to(torch.int32)
    table = torch.empty(B, width, dtype=torch.int32)
    table[:, :common] = ids[:common]
    table[:, common:] = ids[common:common + B * (width - common)].view(B, -1)
    if shared % page:
        for t in (k, v):
            for b in range(1, B):
                t[table[b, common].long(), :shared % page] = t[table[0, common].long(), :shared % page]
    if lens is None:
        lens = shared + torch.randint(T, max(T, own) + 1, (B,), generator=g)
        lens[0] = shared + own
    lens = torch.as_tensor(lens, dtype=torch.int32)
    held = torch.zeros(N, page, dtype=torch.bool)
    for b in range(B):
        n = max(0, int(lens[b]))
        at = torch.arange(n)
        held[table[b].long()[at // page], at % page] = True
    at = torch.arange(shared)
    held[table[0].long()[at // page], at % page] = True
    k[~held], v[~held] = float("nan"), float("nan")
    q = torch.randn(B * T, Hq, D, generator=g)
    return {"q": q.to(device, dtype), "k_cache": k.to(device, dtype), "v_cache": v.to(device, dtype), "kv_lens": lens.to(device),
            "block_table": table.to(device), "shared": shared, "scale": D ** -0.5, "tokens": T}


def page_state(R, W, N, page, seed=0, device="cpu"):
    """Rows of random length with pages of their own, some of which begin with another row's, and a few that are empty; room behind the last
    token in some."""
    g = torch.Generator().manual_seed(seed)
    table = torch.full((R, W), -1, dtype=torch.int32)
    lens, refs = torch.zeros(R, dtype=torch.int32), torch.zeros(N, dtype=torch.int32)
    ids, at = torch.randperm(N, generator=g).tolist(), 0
    for r in range(R):
        kind = int(torch.randint(0, 5, (1,), generator=g))
        if kind == 0:
            continue
        n = int(torch.randint(1, W * page + 1, (1,), generator=g))
        other = int(torch.randint(0, r, (1,), generator=g)) if r and kind in (1, 2) else -1
        common = 0
        if other >= 0 and int(lens[other]) > 0:
            n = min(n, int(lens[other])) if kind == 1 else n
            common = min(-(-n // page), -(-int(lens[other]) // page) if kind == 1 else int(lens[other]) // page)
        held = min(W, -(-n // page) + (kind == 3))
        if at + held - common > N:
            continue
        table[r, :common] = table[other, :common] if common else table[r, :common]
        for w in range(common, held):
            table[r, w] = ids[at]
            at += 1
        lens[r] = n
        for w in range(held):
            refs[table[r, w].long()] += 1
    return table.to(device), lens.to(device), refs.to(device)


def counts_of(table, N):
    """How many table entries hold each page."""
    flat = table.flatten().long()
    return torch.bincount(flat[(flat >= 0) & (flat < N)], minlength=N).to(torch.int32)


def draft_batch(B, K, V, dtype=torch.float32, sampled=True, seed=0, ragged=False, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g) * 2
    near = logits[:, :K] + torch.randn(B, K, V, generator=g) * 0.5
    p, q = torch.softmax(logits, -1).to(dtype), torch.softmax(near, -1).to(dtype)
    drafts = torch.multinomial(q.float().reshape(B * K, V), 1, generator=g).view(B, K) if sampled and K else near.argmax(-1).view(B, K)
    lens = torch.randint(0, K + 1, (B,), generator=g, dtype=torch.int32) if ragged else None
    u = torch.rand(B, K + 1, generator=g)
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    return {"drafts": to(drafts), "target_probs": to(p), "uniform": to(u), "draft_probs": to(q) if sampled else None, "draft_lens": to(lens)}
