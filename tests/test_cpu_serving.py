"""Operators for several continuations of one prompt: their reference semantics, and what they refuse, without a GPU."""
import pytest
import torch

from serving_cases import counts_of, draft_batch, page_state, prefix_batch
from triton_distributed_b200 import ops, ref
from triton_distributed_b200.models import PagePool


def test_shared_prefix_reference_is_paged_attention():
    c = prefix_batch(3, 1, 4, 2, 64, 16, 37, 20, dtype=torch.float32)
    out, lse = ref.shared_prefix_attention_ref(**c)
    want, want_lse = ref.paged_decode_attention_ref(c["q"], c["k_cache"], c["v_cache"], c["kv_lens"], c["block_table"], c["scale"])
    torch.testing.assert_close(out.float(), want, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(lse.float(), want_lse, rtol=1e-5, atol=1e-5)


def test_verify_reference_follows_the_target():
    """Over many draws the first token is distributed as the target says (5 tokens, 20000 draws: a frequency is off by more than
    4.5 standard deviations, 4.5 * sqrt(0.25 / 20000) = 0.016, once in about 1e5 runs; the seed is fixed)."""
    B, V = 20000, 5
    g = torch.Generator().manual_seed(3)
    p, q = torch.softmax(torch.randn(2, V, generator=g) * 1.5, -1), torch.softmax(torch.randn(1, V, generator=g) * 1.5, -1)
    drafts = torch.multinomial(q.expand(B, V), 1, generator=g)
    u = torch.rand(B, 2, generator=g)
    acc, tokens = ref.verify_drafts_ref(drafts, p.expand(B, 2, V), u, q.expand(B, 1, V))
    freq = torch.bincount(tokens[:, 0], minlength=V) / B
    assert (freq - p[0]).abs().max() < 0.016
    assert 0 < int(acc.sum()) < B


@pytest.mark.parametrize("seed", range(6))
def test_page_references_keep_the_counts(seed):
    R, W, N, page = 9, 5, 40, 4
    table, lens, refs = page_state(R, W, N, page, seed)
    assert torch.equal(counts_of(table, N), refs)
    g = torch.Generator().manual_seed(seed)
    src, dst = torch.randint(0, R, (4,), generator=g), torch.randperm(R, generator=g)[:4]
    table, lens, refs = ref.fork_pages_ref(table, lens, refs, src, dst, page)
    assert torch.equal(counts_of(table, N), refs)
    status, table, refs, copies = ref.reserve_pages_ref(table, lens, refs, (torch.rand(R, generator=g) * 4).int(), page)
    assert torch.equal(counts_of(table, N), refs)
    table, lens, refs = ref.trim_pages_ref(table, lens, refs, page, lens - 2)
    assert torch.equal(counts_of(table, N), refs)
    table, refs, moves = ref.compact_pages_ref(table, refs)
    assert torch.equal(counts_of(table, N), refs)
    live = int((refs > 0).sum())
    assert bool((refs[:live] > 0).all())


def _refused(error, call, *a, **kw):
    with pytest.raises(error):
        call(*a, **kw)


def test_shared_prefix_attention_refuses():
    ok = prefix_batch(2, 2, 4, 2, 64, 16, 32, 16)
    call = lambda **kw: ops.shared_prefix_attention(**{**ok, **kw})  # noqa: E731
    _refused(TypeError, call, q=ok["q"].float())
    _refused(TypeError, call, v_cache=ok["v_cache"].to(torch.float16))
    _refused(TypeError, call, kv_lens=ok["kv_lens"].long())
    _refused(TypeError, call, block_table=ok["block_table"].long())
    _refused(ValueError, call, tokens=3)
    _refused(ValueError, call, tokens=0)
    _refused(ValueError, call, scale=0.0)
    _refused(ValueError, call, scale=float("nan"))
    _refused(ValueError, call, shared=-1)
    _refused(ValueError, call, shared=49)                                  # the table has three pages
    _refused(ValueError, call, shared=(1 << 30) + 1)                       # lengths and ranges of keys stay in 32 bits
    _refused(ValueError, call, q=ok["q"][:, :3])                           # three query heads for two of the cache
    _refused(ValueError, call, q=ok["q"][..., :32])
    _refused(ValueError, call, q=ok["q"].transpose(0, 1))
    _refused(ValueError, call, q=ok["q"][:1].expand(4, 4, 64))
    _refused(ValueError, call, kv_lens=ok["kv_lens"][:1])
    _refused(ValueError, call, k_cache=ok["k_cache"][:, ::2], v_cache=ok["v_cache"][:, ::2])
    _refused(ValueError, call, prefix_table=ok["block_table"][0, :1])      # two pages are shared
    _refused(TypeError, call, prefix_table=ok["block_table"][0].long())
    _refused(ValueError, call, out=torch.empty(4, 4, 64))
    wide = prefix_batch(2, 1, 4, 2, 96, 16, 32, 16)
    _refused(ValueError, ops.shared_prefix_attention, **wide)
    if not torch.cuda.is_available():
        _refused(RuntimeError, call)
    else:
        _refused(ValueError, call)   # tensors of the CPU


def test_verify_drafts_refuses():
    ok = draft_batch(2, 3, 11)
    call = lambda **kw: ops.verify_drafts(**{**ok, **kw})  # noqa: E731
    _refused(ValueError, call, drafts=ok["drafts"][:, :2])
    _refused(TypeError, call, drafts=ok["drafts"].int())
    _refused(TypeError, call, uniform=ok["uniform"].double())
    _refused(ValueError, call, uniform=ok["uniform"][:, :3])
    _refused(TypeError, call, draft_probs=ok["draft_probs"].bfloat16())
    _refused(TypeError, call, target_probs=ok["target_probs"].double(), draft_probs=None)
    _refused(ValueError, call, draft_probs=ok["draft_probs"][:, :, :10])
    _refused(TypeError, call, draft_lens=torch.tensor([1, 2]))
    _refused(ValueError, call, draft_lens=torch.tensor([1], dtype=torch.int32))
    _refused(ValueError, call, target_probs=ok["target_probs"].transpose(1, 2).contiguous().transpose(1, 2))
    _refused(ValueError if torch.cuda.is_available() else RuntimeError, call)


def test_page_operators_refuse():
    table, lens, refs = page_state(6, 4, 30, 8)
    caches = [torch.zeros(2, 30, 8, 4), torch.zeros(2, 30, 8, 2)]
    here = ValueError if torch.cuda.is_available() else RuntimeError   # tensors of the CPU, or no GPU
    _refused(TypeError, ops.fork_pages, table.long(), lens, refs, [0], [1], 8)
    _refused(TypeError, ops.fork_pages, table[:, ::2], lens, refs, [0], [1], 8)
    _refused(ValueError, ops.fork_pages, table, lens[:3], refs, [0], [1], 8)
    _refused(ValueError, ops.fork_pages, table, lens, refs, [0, 1], [1], 8)
    _refused(ValueError, ops.fork_pages, table, lens, refs, [[0]], [[1]], 8)
    _refused(ValueError, ops.fork_pages, table, lens, refs, torch.tensor([0.0]), [1], 8)
    _refused(ValueError, ops.fork_pages, table, lens, refs, [0], [1], 0)
    _refused(here, ops.fork_pages, table, lens, refs, [0], [1], 8)
    _refused(ValueError, ops.trim_pages, table, lens, refs, 8, lens[:2])
    _refused(ValueError, ops.trim_pages, table, lens, refs, 8, lens.long())
    _refused(here, ops.trim_pages, table, lens, refs, 8, lens)
    _refused(ValueError, ops.reserve_pages, table, lens, refs, -1, caches, dim=1)
    _refused(ValueError, ops.reserve_pages, table, lens, refs, lens.long(), caches, dim=1)
    _refused(ValueError, ops.reserve_pages, table, lens, refs, 1, [], dim=1)
    _refused(ValueError, ops.reserve_pages, table, lens, refs, 1, caches, dim=2)
    _refused(ValueError, ops.reserve_pages, table, lens, refs, 1, caches, dim=0)                                # two pages for 30 counts
    _refused(ValueError, ops.reserve_pages, table, lens, refs, 1, [caches[0], torch.zeros(2, 30, 4, 4)], dim=1)  # pages of other sizes
    _refused(ValueError, ops.reserve_pages, table, lens, refs, 1, [torch.zeros(2, 30, 8, 8)[..., ::2]], dim=1)
    _refused(here, ops.reserve_pages, table, lens, refs, 1, caches, dim=1)
    _refused(ValueError, ops.compact_pages, table, refs, caches, dim=1, out=(table[:2], refs))
    _refused(here, ops.compact_pages, table, refs, caches, dim=1)
    _refused(ValueError, ops.copy_pages, caches, [0, 1], [2], dim=1)
    _refused(ValueError, ops.copy_pages, caches, [0, 1], [2, 2], dim=1)
    _refused(ValueError, ops.copy_pages, caches, [0, 1], [1, 2], dim=1)
    _refused(ValueError, ops.copy_pages, caches, [0], [30], dim=1)
    _refused(ValueError, ops.copy_pages, caches, [-1], [3], dim=1)
    _refused(ValueError, ops.copy_pages, caches, [0], [3], dim=1, tokens=[9])
    _refused(here, ops.copy_pages, caches, [0], [3], dim=1)


def test_pool_slots():
    pool = PagePool(1, 8, 3, 64, 1, 8, torch.float32, page_size=16, device="cpu")
    pool.block_table[0, :2] = torch.tensor([3, 5])
    pool.kv_lens[:] = torch.tensor([15, 0, 64])
    spare = 8 * 16
    assert pool.slots(3).tolist() == [3 * 16 + 15, 5 * 16, 5 * 16 + 1, spare, spare + 1, spare + 2, spare, spare + 1, spare + 2]


@pytest.mark.parametrize("B,T,heads,kv,shared,own,page", [(1, 1, 8, 8, 0, 1, 64), (256, 1, 8, 1, 131072, 256, 128), (64, 1, 64, 8, 32768, 1024, 64), (3, 8, 28, 4, 100, 50, 44),
                                                          (4, 1, 64, 8, 9000, 10, 16), (1, 300, 4, 4, 5, 1, 8)])
@pytest.mark.parametrize("variant", [None, "warp", "tc"])
def test_prefix_splits_cover_the_keys(B, T, heads, kv, shared, own, page, variant):
    if variant == "tc" and (shared == 0 or page == 44):
        with pytest.raises(ValueError):
            ops.choose_prefix_splits(B, T, heads, kv, shared, own, page, variant=variant)
        return
    tc, prefix, mine = ops.choose_prefix_splits(B, T, heads, kv, shared, own, page, variant=variant)
    assert tc == (variant == "tc") or variant is None
    assert (prefix == 0) == (shared == 0) and 1 <= mine <= 64 and prefix <= 64


def _pool_of_two(free=0):
    """Row 0 holds 28 tokens, row 1 is a fork of it that was cut back to 20: both hold the page of tokens 16 ... 31."""
    pool = PagePool(1, 2 + free, 2, 64, 1, 8, torch.float32, page_size=16, device="cpu")
    pool.block_table[:, :2] = torch.tensor([0, 1])
    pool.kv_lens[:] = torch.tensor([28, 20])
    pool.refs[:2] = 2
    return pool


@pytest.mark.parametrize("counts,free", [([2, 2], 0), ([0, 0], 4), ([2, 0], 0)])
def test_pool_slots_are_in_no_page_that_others_hold(counts, free):
    """A row that got no copy of a page that others hold (too few pages were free, or it asked for none) writes to the spare page."""
    pool = _pool_of_two(free)
    status, table, refs, _ = ref.reserve_pages_ref(pool.block_table, pool.kv_lens, pool.refs, torch.tensor(counts), 16)
    assert status == (1 if any(counts) else 0)
    pool.block_table.copy_(table), pool.refs.copy_(refs)
    spare = (2 + free) * 16
    assert pool.slots(2).tolist() == [spare + 12, spare + 13, spare + 4, spare + 5]


def test_pool_slots_of_a_row_that_pauses():
    """Row 0 goes on in a copy and row 1 pauses: the page is row 1's alone then, and its next slots hold nobody's tokens."""
    pool = _pool_of_two(3)
    status, table, refs, copies = ref.reserve_pages_ref(pool.block_table, pool.kv_lens, pool.refs, torch.tensor([2, 0]), 16)
    pool.block_table.copy_(table), pool.refs.copy_(refs)
    assert status == 0 and copies == [(1, 2, 12)]
    assert pool.slots(2).tolist() == [2 * 16 + 12, 2 * 16 + 13, 16 + 4, 16 + 5]


def test_pool_check_looks_once():
    pool = _pool_of_two()
    for code in (1, 2):
        pool.status.fill_(code)
        with pytest.raises(RuntimeError):
            pool.check()
        pool.check()
    table, lens, refs = page_state(6, 4, 30, 8)
    _refused(ValueError, ops.reserve_pages, table, lens, refs, 1, [torch.zeros(30, 8, 4)], keep=True)   # there is no status to keep


@pytest.mark.parametrize("advanced", [16, 9, 33])
@pytest.mark.parametrize("held", [0, 1])
def test_reserve_reference_leaves_no_gap(held, advanced):
    """A row whose length went on after a reserve that found no room is refused until it is cut back to what it holds."""
    table, refs = torch.full((2, 5), -1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    table[0, :held] = torch.arange(held, dtype=torch.int32)
    table[1, :4 - held] = torch.arange(held, 4, dtype=torch.int32)
    refs[:] = 1
    lens = torch.tensor([16 * held, 64 - 16 * held], dtype=torch.int32)
    asks = torch.tensor([advanced, 0], dtype=torch.int32)
    status, table, refs, _ = ref.reserve_pages_ref(table, lens, refs, asks, 16)
    assert status == 1
    table, lens, refs = ref.trim_pages_ref(table, lens + asks, refs, 16, None, [1])       # advanced unseen; the other row ends
    before = table.clone(), refs.clone()
    status, table, refs, copies = ref.reserve_pages_ref(table, lens, refs, torch.tensor([1, 1]), 16)
    assert status == 3 and not copies and torch.equal(table, before[0]) and torch.equal(refs, before[1])
    assert ref.reserve_pages_ref(table, lens, refs, torch.tensor([0, 1]), 16)[0] == 0     # rows that do not ask are left alone
    table, lens, refs = ref.trim_pages_ref(table, lens, refs, 16, torch.tensor([16 * held]), [0])
    status, table, refs, _ = ref.reserve_pages_ref(table, lens, refs, torch.tensor([1, 1]), 16)
    assert status == 0 and torch.equal(counts_of(table, 4), refs)


def test_pool_check_names_the_gap():
    pool = _pool_of_two()
    pool.status.fill_(3)
    with pytest.raises(RuntimeError, match="last token"):
        pool.check()


@pytest.mark.parametrize("heads,tokens", [(128, 131070), (64, 262140), (43, 262140), (1, 16776960)])
def test_rows_that_no_grid_of_tiles_holds(heads, tokens):
    """Pairs of tiles of 128 // heads tokens are counted by the second dimension of a grid, 65535 at most: more rows go to the warp kernel."""
    choice = lambda n, **kw: ops.choose_prefix_splits(1, n, heads, 1, 1024, n, **kw)[0]  # noqa: E731
    assert choice(tokens) and choice(tokens, variant="tc")
    assert not choice(tokens + 1) and not choice(tokens + 1, variant="warp")
    with pytest.raises(ValueError):
        choice(tokens + 1, variant="tc")


def test_rows_outside_32_bits_stay_outside():
    """Row numbers that 32 bits do not hold name no row, not the one with the same low bits."""
    far = [2**32, 2**32 + 3, -2**32, 2**31, -2**31 - 1, 2**63 - 1, -2**63, -1, 5]
    for rows in (far, torch.tensor(far)):
        got = ops._rows("fork_pages", rows, torch.device("cpu"))
        assert got.dtype == torch.int32 and got[-1] == 5 and bool(((got[:-1] < 0) | (got[:-1] == 2**31 - 1)).all())


@pytest.mark.parametrize("R,N", [(1, 1), (9, 60), (1500, 70000), (2**20, 2**27)])
def test_pages_scratch_holds_both_layouts(R, N):
    """Room: moves (4 words) and plans (4) of the rows, three lists of pages, a count. Compaction: moves (4 words) and three lists of pages, a count."""
    assert ops._pages_scratch(R, N) >= max(8 * R + 3 * N + 1, 7 * N + 1)


@pytest.mark.parametrize("tokens", [1, 3])
def test_pool_prefix_table_outlives_the_first_row(tokens):
    """The row that was forked ends (or is cut back), rows of other prompts that are no longer than the shared keys stand in front: the pages of the
    shared keys come from the first row that reaches beyond them."""
    shared, page = 20, 8
    c = prefix_batch(5, tokens, 4, 2, 64, page, shared, 12, dtype=torch.float32, lens=[30, 25, 0, 26, 30])
    want, _ = ref.shared_prefix_attention_ref(**c)
    pool = PagePool(1, c["k_cache"].shape[0] - 1, 5, 32, 2, 64, torch.float32, page_size=page, device="cpu")
    pool.block_table.copy_(c["block_table"]), pool.kv_lens.copy_(c["kv_lens"])
    pool.block_table[0], pool.kv_lens[0] = -1, 0
    pool.block_table[1, :3], pool.kv_lens[1] = c["block_table"][4, 1:].flip(0), shared + tokens - 2     # another text
    c["block_table"], c["kv_lens"] = pool.block_table, pool.kv_lens
    first = pool.prefix_table(shared, tokens)
    assert first.dtype == torch.int32 and first.shape == (4,) and first.is_contiguous()
    got, _ = ref.shared_prefix_attention_ref(**c, prefix_table=first)
    torch.testing.assert_close(got[2 * tokens:], want[2 * tokens:], rtol=0, atol=0)
    pool.kv_lens.zero_()
    assert pool.prefix_table(shared, tokens).shape == (4,)      # nobody reads it then


@pytest.mark.parametrize("B,T,heads,kv,page,dim", [(1, 1, 8, 8, 64, 128), (2, 1, 32, 8, 16, 128), (16, 1, 64, 8, 64, 128), (24, 5, 40, 8, 16, 128), (48, 3, 14, 2, 32, 64),
                                                   (64, 1, 64, 8, 64, 128), (256, 1, 8, 1, 128, 128), (9, 4, 160, 1, 64, 64)])
@pytest.mark.parametrize("variant", [None, "warp", "tc"])
def test_ranges_of_shared_keys_lie_side_by_side(B, T, heads, kv, page, dim, variant):
    """The ranges as the launch forms them (chunks of whole slices or steps) cover the shared keys once, and none of the tensor-core kernel's is without
    a step of its own where there are as many steps as ranges."""
    if variant == "tc" and heads // kv > 128:
        pytest.skip("refused: a group that no tile holds")
    for shared in (1, 63, 64, 65, 127, 128, 129, 1000, 2048, 7001, 16384, 100003):
        for own in (1, 300, 5000):
            tc, ranges, _ = ops.choose_prefix_splits(B, T, heads, kv, -(-shared // 128) * 128, max(64, -(-own // 64) * 64), page, dim=dim, variant=variant)
            unit = 128 if tc else 64
            chunk = -(-(-(-shared // ranges)) // unit) * unit
            edges = [(min(shared, i * chunk), min(shared, (i + 1) * chunk)) for i in range(ranges)]
            assert edges[0][0] == 0 and edges[-1][1] == shared and all(a[1] == b[0] for a, b in zip(edges, edges[1:]))
            assert 1 <= ranges <= min(64, -(-shared // 128))
