"""Operators for several continuations of one prompt against plain implementations in 64 bits."""
import pytest
import torch

from serving_cases import counts_of, draft_batch, page_state, prefix_batch

pytestmark = pytest.mark.gpu


def _check_attention(c, out, lse, want, want_lse, spread, most=40):
    """`spread`: sum_j w_j |v_j| of every output. The weights are rounded once to the type (half a step, u), their sum is not, the output is rounded
    once: |error| <= u (spread + |out|). Everything else is fp32: products of at most 128 terms of scores below 40 are off by at most
    128 * 2^-24 * 40 / 2 = 1.5e-4, which moves a weight and the log-sum-exp by that much; sums and merges add a few 2^-24 times the number of terms."""
    u, more = torch.finfo(c["q"].dtype).eps / 2, max(1, most / 40)   # (larger scores are off by more in proportion)
    bound = u * (spread + want.abs()) + 4e-4 * more * spread + 1e-6
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max()):.2f} of the bound"
    empty = want_lse == float("-inf")
    assert torch.equal(lse == float("-inf"), empty)
    assert bool((out[empty] == 0).all())
    assert bool(((lse.double() - want_lse)[~empty].abs() <= 3e-4 * more).all())


def _attention_case(c, most=40, **kw):
    from triton_distributed_b200 import ops, ref
    want, want_lse = ref.shared_prefix_attention_ref(**c)
    v = c["v_cache"].abs()
    spread, _ = ref.shared_prefix_attention_ref(**{**c, "v_cache": v})
    out, lse = ops.shared_prefix_attention(**c, return_lse=True, **kw)
    ops.check_pipeline_status()
    _check_attention(c, out, lse, want, want_lse, spread, most)
    return out


@pytest.mark.parametrize("B,T,Hq,Hkv,D,page,shared,own", [
    (1, 1, 1, 1, 64, 16, 1, 1),          # one key of each
    (1, 1, 8, 8, 128, 64, 0, 1),         # nothing shared, one key
    (2, 1, 8, 2, 128, 64, 64, 1),
    (3, 1, 32, 8, 128, 16, 100, 30),     # a page that ends inside a tile
    (5, 3, 14, 2, 64, 32, 777, 90),      # groups of seven, several tokens
    (4, 8, 28, 4, 128, 48, 1000, 61),    # pages that no tile is a multiple of
    (2, 1, 16, 16, 64, 7, 130, 20),      # pages smaller than a slice
    (33, 1, 8, 1, 128, 128, 3000, 200),
    (70, 1, 40, 8, 128, 64, 513, 5),
    (17, 5, 64, 8, 128, 256, 2048, 300),
    (130, 2, 5, 1, 64, 64, 4100, 17),
    (9, 1, 64, 1, 128, 16, 1500, 40),    # 64 heads on one KV head
    (3, 2, 160, 1, 64, 32, 300, 9),      # 160
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("variant", ["warp", "tc"])
def test_shared_prefix_attention(B, T, Hq, Hkv, D, page, shared, own, dtype, variant):
    if variant == "tc" and (shared == 0 or page == 7 or Hq // Hkv > 128):
        pytest.skip("refused: nothing is shared, pages that no tile is made of, or groups that no tile holds")
    _attention_case(prefix_batch(B, T, Hq, Hkv, D, page, shared, own, dtype, seed=B + shared, device="cuda"), variant=variant)


@pytest.mark.parametrize("B,T,Hq,Hkv,D,page,shared", [
    (1, 1, 1, 1, 64, 8, 1), (1, 1, 8, 8, 128, 16, 127), (2, 3, 16, 2, 128, 32, 128), (5, 1, 40, 8, 128, 64, 129), (3, 2, 128, 1, 64, 128, 256),
    (7, 4, 28, 4, 128, 256, 385), (26, 1, 40, 8, 128, 16, 1111), (40, 1, 14, 2, 64, 64, 5000), (300, 1, 8, 1, 128, 128, 640), (25, 5, 5, 1, 64, 384, 1500),
    (128, 1, 2, 2, 128, 8, 3000), (20, 2, 16, 2, 128, 24, 1000), (50, 1, 8, 2, 64, 48, 2900), (9, 3, 8, 1, 128, 96, 777), (40, 1, 6, 1, 64, 200, 1801), (129, 1, 1, 1, 64, 64, 20000), (64, 1, 64, 8, 128, 16, 2047), (1, 1, 48, 1, 128, 64, 4096)])
def test_shared_prefix_attention_tiles(B, T, Hq, Hkv, D, page, shared):
    """The tensor-core kernel at one and at two tiles of rows, full and ragged steps, all page sizes, head groups that do not divide a tile."""
    _attention_case(prefix_batch(B, T, Hq, Hkv, D, page, shared, 20, seed=B, device="cuda"), variant="tc")


@pytest.mark.parametrize("variant", ["warp", "tc"])
def test_lengths_below_zero_hold_nothing(variant):
    c = prefix_batch(24, 3, 8, 2, 64, 64, 200, 40, device="cuda")
    c["kv_lens"][3:6] = torch.tensor([-1, -2**31, -2**31 + 1], device="cuda", dtype=torch.int32)
    out = _attention_case(c, variant=variant)
    assert bool((out[9:18] == 0).all())


@pytest.mark.parametrize("B,Hq,Hkv,page,shared,own", [
    (80, 8, 2, 16, 1000, 5000),     # thousands of own keys for one CTA
    (80, 2, 2, 48, 999, 4700),
    (2, 16, 16, 32, 70001, 30),     # of shared ones
    (1, 16, 16, 24, 50000, 2),      # pages that no slice is made of
])
def test_shared_prefix_attention_of_many_keys_for_one_cta(B, Hq, Hkv, page, shared, own):
    _attention_case(prefix_batch(B, 1, Hq, Hkv, 64, page, shared, own, seed=page, device="cuda"), variant="warp")


@pytest.mark.parametrize("kv_lens", [[3, 700], [0, 64], [63, 65], [1, 1], [2048, 2049]])
@pytest.mark.parametrize("page", [16, 64, 80])
def test_sequences_that_end_before_the_shared_keys_do(kv_lens, page):
    """Short sequences beside ones that reach beyond the shared keys: whose first pages are read depends on the length."""
    for B in (2, 24):
        lens = (kv_lens * B)[:B]
        _attention_case(prefix_batch(B, 1, 8, 2, 64, page, 64, 2100, seed=B, lens=lens, device="cuda"))


@pytest.mark.parametrize("variant", ["warp", "tc"])
@pytest.mark.parametrize("B", [3, 40])
@pytest.mark.parametrize("order", [1, -1, 0])
def test_scores_that_grow_and_fall(B, order, variant):
    """Later keys outweigh the earlier ones step by step (every reference of the softmax is raised), or the first one all others, or all are alike."""
    c = prefix_batch(B, 1, 16, 2, 128, 64, 1500, 40, device="cuda")
    n = 1540
    size = torch.linspace(0.05, 3.0, n, device="cuda")
    if order == -1:
        size = size.flip(0)
    c["q"] = torch.randn(1, 1, 128, device="cuda").expand(B, 16, 128).to(torch.bfloat16).contiguous()   # one direction
    for b in range(B):
        at = torch.arange(int(c["kv_lens"][b]), device="cuda")
        page, off = c["block_table"][b].long()[at // 64], at % 64
        c["k_cache"][page, off] = (c["q"][0, 0].float() * (size[at, None, None] if order else 0.7)).to(torch.bfloat16)
    _attention_case(c, most=50, variant=variant)   # |q|^2 / sqrt(128) * 3 = 34 on average


@pytest.mark.parametrize("variant", ["warp", "tc"])
def test_keys_that_are_no_numbers(variant):
    """A NaN among the keys, or scores of infinity, make what sees them NaN and nothing else."""
    from triton_distributed_b200 import ops
    c = prefix_batch(20, 1, 16, 2, 128, 64, 1000, 40, device="cuda")
    clean = ops.shared_prefix_attention(**c, variant=variant)
    page = c["block_table"][0].long()
    for where, value in ((777, float("nan")), (5, float("inf"))):
        d = {**c, "k_cache": c["k_cache"].clone()}
        d["k_cache"][page[where // 64], where % 64, 1, 3] = value
        out = ops.shared_prefix_attention(**d, variant=variant)
        assert torch.equal(out[:, :8], clean[:, :8])
        s = d["q"][:, 8:, 3].float() * value       # NaN, or infinity of one sign: plus makes the row NaN, minus is a weight of zero
        gone = s.isnan() | (s == float("inf"))
        assert bool(out[:, 8:][gone].isnan().all()) and bool(out[:, 8:][~gone].isfinite().all())


@pytest.mark.parametrize("first,end,value", [(5, 6, float("nan")), (40, 41, float("nan")), (40, 41, float("inf")), (0, 40, float("inf")),
                                              (0, 128, float("inf")), (128, 256, float("inf")), (0, 1000, float("inf"))])
@pytest.mark.parametrize("B", [4, 40])
def test_first_keys_that_are_no_numbers(B, first, end, value):
    """The first keys give the softmax on the tensor cores its reference: none of them, some, whole steps or all shared keys may have scores of minus
    infinity (for the other half of the rows plus infinity, which like NaN makes a row NaN)."""
    from triton_distributed_b200 import ops, ref
    c = prefix_batch(B, 1, 16, 2, 128, 64, 1000, 40, seed=first + end, device="cuda")
    page, at = c["block_table"][0].long(), torch.arange(first, end, device="cuda")
    c["k_cache"][page[at // 64], at % 64, 1, 3] = value
    want, want_lse = ref.shared_prefix_attention_ref(**c)
    spread, _ = ref.shared_prefix_attention_ref(**{**c, "v_cache": c["v_cache"].abs()})
    out, lse = ops.shared_prefix_attention(**c, return_lse=True, variant="tc")
    ops.check_pipeline_status()
    s = c["q"][..., 3].float() * value
    gone = s.isnan() | (s == float("inf"))
    gone[..., :8] = False                      # the other KV head's keys are numbers
    assert bool(gone.any()) and bool(out[gone].isnan().all())
    out, want, spread = (x.masked_fill(gone[..., None], 0) for x in (out, want, spread))
    lse, want_lse = (x.masked_fill(gone, 0) for x in (lse, want_lse))
    _check_attention(c, out, lse, want, want_lse, spread)


@pytest.mark.parametrize("T,shared", [(1, 200), (4, 200), (3, 64)])
@pytest.mark.parametrize("B", [6, 150])
def test_shared_prefix_attention_of_short_rows(T, shared, B):
    """Rows of the batch without a sequence, sequences shorter than the shared keys, fewer keys than new tokens."""
    lens = [shared + 9, 0, shared - 1, T - 1, shared + T - 1, 5] + [shared + i % 9 for i in range(6, B)]
    c = prefix_batch(B, T, 16, 2, 128, 16, shared, 9, lens=lens, device="cuda")
    for variant in ("warp", "tc"):
        _attention_case(c, variant=variant)


def test_shared_prefix_attention_of_an_own_table_and_strided_rows():
    c = prefix_batch(4, 2, 8, 2, 128, 32, 320, 40, device="cuda")
    plain = _attention_case(c)
    table = c["block_table"][0, :10].clone()
    c["block_table"][:, :10] = 10 ** 6       # nobody's table is read for the shared keys
    from triton_distributed_b200 import ops
    torch.testing.assert_close(ops.shared_prefix_attention(**c, prefix_table=table), plain, rtol=0, atol=0)
    wide = torch.randn(8, 12, 128, device="cuda", dtype=torch.bfloat16)   # q as columns of a wider product
    wide[:, :8] = c["q"]
    out = torch.full_like(c["q"], float("nan"))
    got = ops.shared_prefix_attention(**{**c, "q": wide[:, :8]}, prefix_table=table, out=out, max_kv_len=360)
    assert got is out
    wide_table = torch.cat([c["block_table"], c["block_table"]], 1)[:, :c["block_table"].shape[1]]   # rows further apart than they are long
    torch.testing.assert_close(ops.shared_prefix_attention(**{**c, "block_table": wide_table}, prefix_table=table, max_kv_len=360), out, rtol=0, atol=0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_later_draft_holds_stays_there(dtype, bad):
    """Values (and keys) of a drafted token that are not finite reach the tokens that see it, and no others."""
    c = prefix_batch(3, 4, 8, 2, 128, 16, 50, 14, dtype, lens=[60, 64, 55], device="cuda")
    from triton_distributed_b200 import ops
    clean = ops.shared_prefix_attention(**c).view(3, 4, 8, 128)
    page = c["block_table"][1, 62 // 16].long()     # the third of the second sequence's four tokens
    c["v_cache"][page, 62 % 16, 1, 17] = bad
    out = ops.shared_prefix_attention(**c).view(3, 4, 8, 128)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[1, 2:, 4:, 17] = True
    assert torch.equal(out[~hit], clean[~hit])
    assert not bool(out[hit].isfinite().any())


def test_pages_outside_the_cache_count_as_zeros():
    c = prefix_batch(3, 1, 8, 2, 64, 16, 70, 30, lens=[100, 96, 95], device="cuda")
    c["block_table"][1, 5] = c["k_cache"].shape[0] + 5
    c["block_table"][2, 5] = -7
    c["block_table"][0, 2] = -1     # (for all: the shared keys are read through the first table)
    c["block_table"][1, 2] = c["block_table"][2, 2] = 10 ** 9
    for variant in ("warp", "tc"):
        _attention_case(c, variant=variant)


def test_shared_prefix_attention_offsets_beyond_32_bits():
    """Pages whose elements lie behind 2^31: a cache of 4.6 GB for keys and values each (only the pages in use are looked at)."""
    N, page, Hkv, D = 140000, 128, 1, 128
    k = torch.empty(N, page, Hkv, D, device="cuda", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    small = prefix_batch(3, 1, 8, 1, 128, 128, 300, 100, device="cuda")
    n = small["k_cache"].shape[0]
    k[-n:], v[-n:] = small["k_cache"], small["v_cache"]
    from triton_distributed_b200 import ops
    for variant in ("warp", "tc"):
        want = ops.shared_prefix_attention(**small, variant=variant)
        got = ops.shared_prefix_attention(**{**small, "k_cache": k, "v_cache": v, "block_table": small["block_table"] + (N - n)}, variant=variant)
        assert torch.equal(got, want)


def _same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b.cpu()), (a, b)


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 7), (3, 0, 100), (2, 40, 33), (5, 3, 32003), (40, 2, 1001), (160, 1, 300), (2, 5, 151936)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sampled,ragged", [(True, False), (False, True)])
def test_verify_drafts(B, K, V, dtype, sampled, ragged):
    from triton_distributed_b200 import ops, ref
    c = draft_batch(B, K, V, dtype, sampled, seed=V + K, ragged=ragged)
    _same(ops.verify_drafts(**{k: None if t is None else t.cuda() for k, t in c.items()}), ref.verify_drafts_ref(**c))


def test_verify_drafts_edges():
    """Numbers zero and next to one, drafts outside the vocabulary, rows without a weight, values that are no probabilities, a target equal to the
    draft, one certain token."""
    from triton_distributed_b200 import ops, ref
    B, K, V = 12, 3, 5000
    c = draft_batch(B, K, V, seed=5)
    below_one = 1 - 2.0 ** -24
    c["uniform"][0], c["uniform"][1] = 0.0, below_one
    c["drafts"][2, 1], c["drafts"][3, 0] = V, -1
    c["target_probs"][4] = 0
    c["target_probs"][5, :, ::2] = float("nan")
    c["draft_probs"][5, :, ::3] = float("inf")
    c["target_probs"][6, :, 7], c["target_probs"][6, :, 11] = -1.0, float("inf")
    c["draft_probs"][7] = c["target_probs"][7, :K]
    c["target_probs"][8] = 0
    c["target_probs"][8, :, 4999] = 1
    c["drafts"][8] = 4999
    c["draft_probs"][9] = 1.0                       # above the target everywhere: nothing is left at the refused place
    c["uniform"][9, :K], c["uniform"][9, K] = below_one, 0.0
    c["target_probs"][10] = 2.0 ** -149             # the smallest number of 32 bits
    c["uniform"][11, K] = 1.0                       # not below one: the last token with a weight
    for probs in (c["draft_probs"], None):
        c["draft_probs"] = probs
        want = ref.verify_drafts_ref(**c)
        _same(ops.verify_drafts(**{k: None if t is None else t.cuda() for k, t in c.items()}), want)
        assert int(want[1][4, 0]) == -1


def test_verify_drafts_strided():
    from triton_distributed_b200 import ops, ref
    c = draft_batch(6, 3, 999, seed=9)
    want = ref.verify_drafts_ref(**c)
    g = {k: None if t is None else t.cuda() for k, t in c.items()}
    wide = torch.full((4, 6, 1003), float("nan"), device="cuda")       # places first, rows longer than the vocabulary
    wide[:, :, 1:1000] = g["target_probs"].transpose(0, 1)
    g["target_probs"] = wide[:, :, 1:1000].transpose(0, 1)
    g["draft_probs"] = g["draft_probs"].transpose(0, 1).contiguous().transpose(0, 1)
    _same(ops.verify_drafts(**g), want)
    g["draft_probs"] = g["draft_probs"][:1, :1].expand(6, 3, 999)      # one distribution for all
    c["draft_probs"] = c["draft_probs"][:1, :1].expand(6, 3, 999)
    _same(ops.verify_drafts(**g), ref.verify_drafts_ref(**c))


PAGES = [(1, 1, 2, 1), (9, 5, 60, 4), (40, 12, 300, 16), (300, 6, 2500, 8), (1500, 3, 70000, 16)]


def _caches(layers, N, page, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(layers, N, page, 2, 24, device="cuda", generator=g).to(dtype), torch.randn(layers, N, page, 5, device="cuda", generator=g).to(dtype)]


@pytest.mark.parametrize("R,W,N,page", PAGES)
@pytest.mark.parametrize("seed", [0, 1])
def test_fork_and_trim_pages(R, W, N, page, seed):
    from triton_distributed_b200 import ops, ref
    table, lens, refs = page_state(R, W, N, page, seed)
    g = torch.Generator().manual_seed(seed)
    n = max(1, R // 2)
    src, dst = torch.randint(-1, R + 1, (n,), generator=g), torch.randint(-1, R + 1, (n,), generator=g)   # some out of range, some named twice
    want = ref.fork_pages_ref(table, lens, refs, src, dst, page)
    got = [t.cuda() for t in (table, lens, refs)]
    ops.fork_pages(*got, src.cuda() if seed else src.tolist(), dst.int().cuda(), page)
    _same(got, want)
    cut = torch.randint(-2, W * page + 2, (R,), generator=g, dtype=torch.int32)
    want = ref.trim_pages_ref(*want, page, cut)
    ops.trim_pages(*got, page, cut.cuda())
    _same(got, want)
    rows = [0, R - 1, 0, R, -1]
    want = ref.trim_pages_ref(*want, page, None, rows)
    ops.trim_pages(*got, page, None, rows)
    _same(got, want)
    assert torch.equal(counts_of(got[0].cpu(), N), got[2].cpu())


def test_fork_exchanges_rows():
    from triton_distributed_b200 import ops
    table, lens, refs = (t.cuda() for t in page_state(9, 5, 60, 4, 3))
    old = table.clone(), lens.clone(), refs.clone()
    ops.trim_pages(table, lens, refs, 4, lens.clone())     # room behind the last token is not forked
    trimmed = table.clone()
    ops.fork_pages(table, lens, refs, list(range(9)), list(range(8, -1, -1)), 4)
    assert torch.equal(table, trimmed.flip(0)) and torch.equal(lens, old[1].flip(0))
    ops.fork_pages(table, lens, refs, [], [], 4)


@pytest.mark.parametrize("more", [0, 300])
def test_fork_pairs_outside_the_table_do_not_count(more):
    """A pair whose source is outside the table is as if it were not there: the next one of its destination counts. (Few pairs, and many.)"""
    from triton_distributed_b200 import ops, ref
    table, lens, refs = page_state(9, 5, 60, 4, 3)
    src, dst = [-1] * more + [-1, 3, 9, 2, 4, 5], [8] * more + [0, 0, 1, 1, 1, -1]
    want = ref.fork_pages_ref(table, lens, refs, src, dst, 4)
    assert not torch.equal(want[0], table)
    got = [t.cuda() for t in (table, lens, refs)]
    ops.fork_pages(*got, src, dst, 4)
    _same(got, want)


def test_lengths_that_no_table_holds():
    """The largest int32 as a length of a row, and as a length to keep: all pages of the table, and nothing outside it is touched."""
    from triton_distributed_b200 import ops, ref
    most = 2**31 - 1
    table, lens, refs = page_state(9, 5, 60, 4, 3)
    lens[4] = most
    got = [t.cuda() for t in (table, lens, refs)]
    want = ref.fork_pages_ref(table, lens, refs, [4, 5], [0, 1], 4)
    ops.fork_pages(*got, [4, 5], [0, 1], 4)
    _same(got, want)
    keep = torch.tensor([most, most, 7, -1, most - 1, most, 3, 0, most], dtype=torch.int32)
    want = ref.trim_pages_ref(*want, 4, keep)
    ops.trim_pages(*got, 4, keep.cuda())
    _same(got, want)
    assert int(ops.reserve_pages(*got, 1, [torch.zeros(60, 4, 1, device="cuda")])) == 2
    _same(got, want)


@pytest.mark.parametrize("R,W,N,page", PAGES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
def test_reserve_pages(R, W, N, page, dtype):
    from triton_distributed_b200 import ops, ref
    table, lens, refs = page_state(R, W, N, page, 1)
    lens = torch.minimum(lens, torch.full_like(lens, W * page - 3)).clamp_min(0)   # room in the table for all
    table, lens, refs = ref.trim_pages_ref(table, lens, refs, page, lens) if R < 1000 else (table, lens, refs)
    g = torch.Generator().manual_seed(2)
    src, dst = torch.randint(0, R, (R // 2,), generator=g), torch.randperm(R, generator=g)[:R // 2]
    table, lens, refs = ref.fork_pages_ref(table, lens, refs, src, dst, page)
    counts = torch.randint(0, 4, (R,), generator=g, dtype=torch.int32)
    caches = _caches(2, N if N < 5000 else 3000, page, dtype) if N < 5000 else None
    if caches is None:   # the tables alone are large
        caches = [torch.zeros(N, page, 1, device="cuda", dtype=torch.uint8)]
    dim = 0 if N >= 5000 else 1
    before = [t.clone() for t in caches]
    for count in (counts, 2):
        status, want_table, want_refs, copies = ref.reserve_pages_ref(table, lens, refs, count, page)
        got = [t.cuda() for t in (table, lens, refs)]
        now = [t.clone() for t in before]
        st = ops.reserve_pages(*got, count.cuda() if isinstance(count, torch.Tensor) else count, now, dim=dim)
        assert int(st) == status
        _same(got, (want_table, lens, want_refs))
        for t, old in zip(now, before):
            want = old.clone()
            for a, b, n in copies:
                want.select(dim, b).narrow(dim, 0, n).copy_(old.select(dim, a).narrow(dim, 0, n))
            assert torch.equal(t, want)


def test_reserve_pages_for_prompts():
    """Many pages for some of the rows, more rows than are remembered among them."""
    from triton_distributed_b200 import ops, ref
    R, W, N, page = 90, 700, 60000, 4
    table, lens, refs = torch.full((R, W), -1, dtype=torch.int32), torch.zeros(R, dtype=torch.int32), torch.zeros(N, dtype=torch.int32)
    refs[torch.randperm(N)[:200]] = 1          # pages of others
    counts = torch.tensor([2000 + 7 * r if r % 5 else r for r in range(R)], dtype=torch.int32)
    status, want_table, want_refs, _ = ref.reserve_pages_ref(table, lens, refs, counts, page)
    got = [t.cuda() for t in (table, lens, refs)]
    st = ops.reserve_pages(*got, counts.cuda(), [torch.zeros(N, page, 1, device="cuda", dtype=torch.uint8)])
    assert int(st) == status == 0
    _same(got, (want_table, lens, want_refs))


def test_reserve_pages_without_pages():
    from triton_distributed_b200 import ops
    caches = [torch.arange(6 * 4, device="cuda", dtype=torch.float32).view(6, 4, 1)]
    table = torch.tensor([[0, 1, -1], [0, 1, -1], [2, -1, -1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([6, 6, 4], dtype=torch.int32, device="cuda")
    refs = torch.tensor([2, 2, 1, 1, 1, 0], dtype=torch.int32, device="cuda")   # one page is free: two are needed
    state = [t.clone() for t in (table, lens, refs, caches[0])]
    assert int(ops.reserve_pages(table, lens, refs, 1, caches)) == 1
    assert all(torch.equal(a, b) for a, b in zip((table, lens, refs, caches[0]), state))
    assert int(ops.reserve_pages(table, lens, refs, 9, caches)) == 2            # longer than a row of the table
    assert all(torch.equal(a, b) for a, b in zip((table, lens, refs, caches[0]), state))
    one = torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda")
    assert int(ops.reserve_pages(table, lens, refs, one, caches)) == 0          # one copy is enough: the first row keeps the page
    assert table.tolist() == [[0, 1, -1], [0, 5, -1], [2, -1, -1]] and refs.tolist() == [2, 1, 1, 1, 1, 1]
    assert caches[0][5].flatten().tolist() == [4.0, 5.0, 22.0, 23.0]
    assert int(ops.reserve_pages(table, lens, refs, torch.zeros_like(one), caches)) == 0


@pytest.mark.parametrize("R,W,N,page", PAGES)
@pytest.mark.parametrize("inplace", [True, False])
def test_compact_pages(R, W, N, page, inplace):
    from triton_distributed_b200 import ops, ref
    table, lens, refs = page_state(R, W, N, page, 4)
    want_table, want_refs, moves = ref.compact_pages_ref(table, refs)
    caches = _caches(3, N, page, torch.float16) if N < 5000 else [torch.randint(0, 255, (1, N, page, 3), device="cuda", dtype=torch.uint8)]
    before = [t.clone() for t in caches]
    a, b = table.cuda(), refs.cuda()
    got = ops.compact_pages(a, b, caches, dim=1, out=(a, b) if inplace else None)
    _same(got, (want_table, want_refs))
    if not inplace:
        _same((a, b), (table, refs))
    if moves:
        src, dst = (torch.tensor(x, device="cuda") for x in zip(*moves))
        for t in before:
            t[:, dst] = t[:, src]
    for t, old in zip(caches, before):
        assert torch.equal(t, old)


@pytest.mark.parametrize("shape,dim,dtype", [((20, 4, 3), 0, torch.uint8), ((20, 7, 5), 0, torch.bfloat16), ((3, 20, 16, 2, 64), 1, torch.float16),
                                             ((2, 20, 64, 8, 128), 1, torch.bfloat16), ((20, 3, 2), 0, torch.float64)])
def test_copy_pages(shape, dim, dtype):
    from triton_distributed_b200 import ops
    many = [(torch.rand(shape, device="cuda") * 200).to(dtype) for _ in range(60 if len(shape) == 3 else 2)]   # more tensors than a launch takes
    before = [t.clone() for t in many]
    src, dst, n = [3, 3, 19, 0], [1, 2, 4, 7], [shape[dim + 1], 1, 0, 2]
    ops.copy_pages(many, src, dst, dim, n)
    for t, old in zip(many, before):
        for a, b, k in zip(src, dst, n):
            old.select(dim, b).narrow(dim, 0, k).copy_(old.select(dim, a).narrow(dim, 0, k))
        assert torch.equal(t, old)
    ops.copy_pages(many, [3], [1], dim)
    assert torch.equal(many[0].select(dim, 1), many[0].select(dim, 3))
    ops.copy_pages(many, [], [], dim)


def test_pages_of_layers_that_lie_apart():
    """Keys and values of a layer side by side, [layers, 2, pages, ...]: the pages of a layer are contiguous, the layers are not."""
    from triton_distributed_b200 import ops
    both = torch.randn(3, 2, 9, 4, 2, 8, device="cuda")
    want = both.clone()
    want[:, :, 7, :3] = want[:, :, 2, :3]
    ops.copy_pages([both[:, 0], both[:, 1]], [2], [7], dim=1, tokens=[3])
    assert torch.equal(both, want)


def _write(pool, layer, slots, k, v):
    pool.layer(layer)[0].view(-1, pool.kv_heads, pool.head_dim)[slots] = k
    pool.layer(layer)[1].view(-1, pool.kv_heads, pool.head_dim)[slots] = v


def test_a_prompt_continued_by_drafts():
    """The operators as they are used together: a prompt is prefilled once and forked, all rows draft, write, attend and are cut back to what was accepted;
    rows end, the cache is compacted, the rest goes on. Attention is that of every row's own text, kept apart on the side."""
    from triton_distributed_b200 import ops
    from triton_distributed_b200.models import PagePool
    torch.manual_seed(0)
    R, K, Hkv, Hq, D, page, V = 6, 3, 2, 8, 128, 16, 700
    pool = PagePool(2, 70, R, 400, Hkv, D, page_size=page)
    text = [[None, None] for _ in range(R)]        # per row and layer: keys and values of its tokens
    prompt = 75
    count = torch.zeros(R, dtype=torch.int32, device="cuda")
    count[0] = prompt
    pool.reserve(count)
    slots = pool.slots(prompt)[:prompt]
    for i in range(2):
        kv = torch.randn(2, prompt, Hkv, D, device="cuda", dtype=torch.bfloat16)
        _write(pool, i, slots, *kv)
        text[0][i] = kv
    pool.advance(count)
    live = list(range(R))
    pool.fork([0] * (R - 1), list(range(1, R)))
    for r in range(1, R):
        text[r] = list(text[0])
    assert int((pool.refs > 0).sum()) == 5         # one copy of the prompt
    T = K + 1
    for step in range(12):
        active = torch.zeros(R, dtype=torch.int32, device="cuda")
        active[live] = T
        start = pool.kv_lens.clone()
        pool.reserve(active)
        slots = pool.slots(T)
        pool.advance(active)
        for i in range(2):
            new = torch.randn(2, R, T, Hkv, D, device="cuda", dtype=torch.bfloat16)
            _write(pool, i, slots, *new.view(2, R * T, Hkv, D))
            q = torch.randn(R * T, Hq, D, device="cuda", dtype=torch.bfloat16)
            first = pool.block_table[live[0]].contiguous()
            out = ops.shared_prefix_attention(q, *pool.layer(i), pool.kv_lens, pool.block_table, prompt, D ** -0.5, tokens=T, prefix_table=first)
            for r in range(R):
                if r not in live:
                    assert bool((out[r * T:(r + 1) * T] == 0).all())
                    continue
                text[r][i] = torch.cat([text[r][i], new[:, r]], 1)
                k, v = text[r][i].float()
                n = k.shape[0]
                s = torch.einsum("tkgd,nkd->tkgn", q[r * T:(r + 1) * T].float().view(T, Hkv, Hq // Hkv, D), k) * D ** -0.5
                s.masked_fill_(torch.arange(n, device="cuda") > (n - T + torch.arange(T, device="cuda"))[:, None, None, None], float("-inf"))
                want = torch.einsum("tkgn,nkd->tkgd", s.softmax(-1), v).reshape(T, Hq, D)
                # rounded weights and output: 2^-8 (spread + |out|) with |v| below 5.5 and the weights' sum one
                torch.testing.assert_close(out[r * T:(r + 1) * T].float(), want, rtol=2 ** -7, atol=2 ** -6)
        d = draft_batch(R, K, V, seed=step, device="cuda")
        accepted, tokens = ops.verify_drafts(**d)
        keep = start + accepted + 1                # the token before the drafts, and the drafts that stand
        pool.trim(torch.where(active > 0, keep, -1).int())
        for r in live:
            text[r] = [t[:, :int(keep[r])] for t in text[r]]
        assert torch.equal(counts_of(pool.block_table.cpu(), 70), pool.refs.cpu())
        if step in (3, 6):
            pool.free([live.pop(1)])
            pool.compact()
            n = int((pool.refs > 0).sum())
            assert bool((pool.refs[:n] > 0).all()) and int(pool.block_table.max()) < n
        if step == 8:                              # one of them branches again, from where it stands
            pool.fork([live[1]], [1])
            text[1] = list(text[live[1]])
            live.append(1)
    with pytest.raises(RuntimeError):
        pool.reserve(399)
    with pytest.raises(RuntimeError):
        pool.reserve(torch.full((R,), 250, dtype=torch.int32, device="cuda"))


def test_a_captured_step():
    """A step in a graph, replayed on other data and next to a second graph and eager calls; results are those of the step alone."""
    from triton_distributed_b200 import ops
    from triton_distributed_b200.models import PagePool
    R, page, K = 4, 16, 2

    def make(seed):
        torch.manual_seed(seed)
        pool = PagePool(1, 40, R, 200, 2, 64, page_size=page)
        pool.k_cache.normal_(), pool.v_cache.normal_()
        n = torch.zeros(R, dtype=torch.int32, device="cuda")
        n[0] = 70
        pool.reserve(n), pool.advance(n)
        pool.fork([0, 0, 0], [1, 2, 3])
        return {"pool": pool, "q": torch.randn(R * 3, 8, 64, device="cuda", dtype=torch.bfloat16), **draft_batch(R, K, 300, seed=seed, device="cuda")}

    def step(s):
        pool = s["pool"]
        pool.reserve(3, check=False)
        pool.advance(3)
        out = ops.shared_prefix_attention(s["q"], *pool.layer(0), pool.kv_lens, pool.block_table, 70, 0.125, tokens=3)
        accepted, tokens = ops.verify_drafts(s["drafts"], s["target_probs"], s["uniform"], s["draft_probs"])
        pool.trim(pool.kv_lens - K + accepted)
        return out, accepted, tokens

    eager, results = [make(0), make(1)], []
    for s in eager:
        results.append([[t.clone() for t in step(s)] + [s["pool"].kv_lens.clone(), s["pool"].block_table.clone()] for _ in range(4)])
    states, graphs, outs = [make(0), make(1)], [], []
    for s in states:
        keep = [t.clone() for t in (s["pool"].block_table, s["pool"].kv_lens, s["pool"].refs)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        for t, old in zip((s["pool"].block_table, s["pool"].kv_lens, s["pool"].refs), keep):
            t.copy_(old)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s))
        graphs.append(g)
    third = make(2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(4):
        for j in (0, 1):
            with torch.cuda.stream(streams[j]):
                graphs[j].replay()
        if i == 0:
            step(third)
        torch.cuda.synchronize()
        for j in (0, 1):
            got = [*outs[j], states[j]["pool"].kv_lens, states[j]["pool"].block_table]
            assert all(torch.equal(a, b) for a, b in zip(got, results[j][i])), (i, j)
    ops.check_pipeline_status()


def test_two_calls_on_two_streams():
    from triton_distributed_b200 import ops
    cases = [prefix_batch(40, 1, 32, 8, 128, 64, 3000, 100, seed=s, device="cuda") for s in (0, 1)]
    want = [ops.shared_prefix_attention(**c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for j in (0, 1):
            with torch.cuda.stream(streams[j]):
                got[j].append(ops.shared_prefix_attention(**cases[j]))
    torch.cuda.synchronize()
    for j in (0, 1):
        assert all(torch.equal(g, want[j]) for g in got[j])


def test_empty_calls():
    from triton_distributed_b200 import ops
    k = torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    out = ops.shared_prefix_attention(torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16), k, k, z(0), z(0, 3), 0, 1.0)
    assert out.shape == (0, 4, 64)
    c = draft_batch(0, 2, 5, sampled=False, device="cuda")
    accepted, tokens = ops.verify_drafts(**c)
    assert accepted.shape == (0,) and tokens.shape == (0, 3)


def test_rows_without_a_copy_write_nobodys_tokens():
    """Rows of different length that hold one page: a step that finds no page for the copies, and a step in which both pause, leave the tokens of all rows
    as they were, captured and replayed too."""
    from triton_distributed_b200.models import PagePool
    pool = PagePool(1, 2, 2, 64, 1, 8, torch.float32, page_size=16)
    n = torch.tensor([28, 0], dtype=torch.int32, device="cuda")
    pool.reserve(n)
    _write(pool, 0, pool.slots(28)[:28], *torch.randn(2, 28, 1, 8, device="cuda"))
    pool.advance(n)
    pool.fork([0], [1])
    pool.trim(torch.tensor([28, 20], dtype=torch.int32, device="cuda"))
    assert pool.refs.tolist() == [2, 2]
    tokens, state = pool.k_cache[:, :2].clone(), [t.clone() for t in (pool.block_table, pool.refs)]

    def step(count):
        pool.reserve(count, check=False)
        _write(pool, 0, pool.slots(2), torch.full((4, 1, 8), 7.0, device="cuda"), torch.full((4, 1, 8), 7.0, device="cuda"))

    counts = [torch.tensor(c, dtype=torch.int32, device="cuda") for c in ([2, 2], [2, 0], [0, 0])]
    for count in counts:
        step(count)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(counts[0])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(pool.k_cache[:, :2], tokens)
    _same((pool.block_table, pool.refs), state)


def test_a_reserve_that_failed_is_remembered():
    """The outcome of an unchecked reserve (of a captured step) is there after later ones that found room, and is gone once it has been looked at."""
    from triton_distributed_b200 import ops
    from triton_distributed_b200.models import PagePool
    pool = PagePool(1, 3, 2, 64, 1, 8, torch.float32, page_size=16)
    g = torch.cuda.CUDAGraph()
    count = torch.tensor([16, 48], dtype=torch.int32, device="cuda")
    pool.reserve(torch.zeros_like(count))
    with torch.cuda.graph(g):
        pool.reserve(count, check=False)
    for counts, code, after in (([16, 48], 1, 1), ([16, 0], 0, 1), ([16, 64], 1, 1), ([65, 0], 2, 2), ([16, 0], 0, 2)):
        count.copy_(torch.tensor(counts, dtype=torch.int32))
        g.replay()
        assert int(pool.status) == after
        alone = ops.reserve_pages(pool.block_table.clone(), pool.kv_lens, pool.refs.clone(), count, (pool.k_cache.clone(), pool.v_cache.clone()), dim=1)
        assert int(alone) == code
    with pytest.raises(RuntimeError, match="max_length"):
        pool.check()
    pool.check()
    pool.reserve(count)
    with pytest.raises(RuntimeError, match="free pages"):
        pool.reserve(torch.tensor([16, 64], dtype=torch.int32, device="cuda"))
    pool.reserve(count)


@pytest.mark.parametrize("advanced", [16, 9, 33])
@pytest.mark.parametrize("held", [0, 1])
def test_rows_that_went_on_without_room(held, advanced):
    """A row whose length was raised after a reserve that found no room gets no pages behind the gap; cut back to what it holds it goes on."""
    from triton_distributed_b200 import ops
    from triton_distributed_b200.models import PagePool
    pool = PagePool(1, 4, 2, 80, 1, 8, torch.float32, page_size=16)
    first = torch.tensor([16 * held, 64 - 16 * held], dtype=torch.int32, device="cuda")
    pool.reserve(first), pool.advance(first)
    asks = torch.tensor([advanced, 0], dtype=torch.int32, device="cuda")
    pool.reserve(asks, check=False)
    pool.advance(asks)
    pool.free([1])
    with pytest.raises(RuntimeError, match="free pages"):
        pool.check()
    state = [t.clone() for t in (pool.block_table, pool.kv_lens, pool.refs)]
    with pytest.raises(RuntimeError, match="last token"):
        pool.reserve(1)
    _same((pool.block_table, pool.kv_lens, pool.refs), state)
    assert int(ops.reserve_pages(*state, 80, (pool.k_cache, pool.v_cache), dim=1)) == 2      # a row of the table is too short in the first place
    pool.reserve(torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    pool.trim(torch.tensor([16 * held], dtype=torch.int32, device="cuda"), [0])
    pool.reserve(1)
    assert torch.equal(counts_of(pool.block_table.cpu(), 4), pool.refs.cpu())


def test_more_rows_than_a_grid_of_tiles_holds():
    """131071 sequences with 128 query heads on one KV head: a tile holds one token, and there are more pairs of tiles than a grid counts."""
    from triton_distributed_b200 import ops, ref
    B, D, page = 131071, 64, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(9, page, 1, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    table = torch.zeros(B, 2, dtype=torch.int32, device="cuda")
    table[:, 1] = 1 + torch.arange(B, device="cuda") % 8
    lens = (65 + torch.arange(B, device="cuda") % 50).int()
    q = torch.randn(B, 128, D, device="cuda", generator=g, dtype=torch.bfloat16)
    out, lse = ops.shared_prefix_attention(q, k, v, lens, table, 64, 0.125, return_lse=True)
    some = torch.tensor([0, 1, 4097, 65534, 65535, 65536, B - 2, B - 1], device="cuda")
    c = {"q": q[some], "k_cache": k, "v_cache": v, "kv_lens": lens[some], "block_table": table[some], "shared": 64, "scale": 0.125}
    want, want_lse = ref.shared_prefix_attention_ref(**c)
    spread, _ = ref.shared_prefix_attention_ref(**{**c, "v_cache": v.abs()})
    _check_attention(c, out[some], lse[some], want, want_lse, spread)


def test_rows_that_32_bits_do_not_hold_are_skipped():
    from triton_distributed_b200 import ops, ref
    state = page_state(9, 5, 60, 4, 3)
    got = [t.cuda() for t in state]
    far = torch.tensor([2**32 + 3, 0, 2**32, -2**32 + 1], device="cuda")
    ops.fork_pages(*got, far, [1, 2**32 + 2, 4, 5], 4)
    ops.fork_pages(*got, [2**32] * 300, [7] * 300, 4)
    ops.trim_pages(*got, 4, None, far[[0, 2, 3]])
    _same(got, state)
    ops.trim_pages(*got, 4, None, far)
    _same(got, ref.trim_pages_ref(*state, 4, None, [0]))


def test_samples_go_on_when_the_first_row_has_ended():
    """Row 0, whose prompt the others share, ends and the pages are compacted: in a captured step too, the others attend as they would alone."""
    from triton_distributed_b200 import ops, ref
    from triton_distributed_b200.models import PagePool
    torch.manual_seed(4)
    pool = PagePool(1, 40, 20, 256, 2, 128, page_size=16)
    n = torch.zeros(20, dtype=torch.int32, device="cuda")
    n[0] = 150
    pool.reserve(n)
    pool.k_cache.normal_(), pool.v_cache.normal_()
    pool.advance(n)
    pool.fork([0] * 19, list(range(1, 20)))
    pool.reserve(1), pool.advance(1)
    q = torch.randn(20, 16, 128, device="cuda", dtype=torch.bfloat16)
    call = lambda: ops.shared_prefix_attention(q, *pool.layer(0), pool.kv_lens, pool.block_table, 150, 128 ** -0.5, prefix_table=pool.prefix_table(150))  # noqa: E731
    before = call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for gone in ([0], [1, 2]):
        pool.free(gone)
        pool.compact()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[3:], before[3:]) and bool((out[gone] == 0).all())
    want, _ = ref.shared_prefix_attention_ref(q, *pool.layer(0), pool.kv_lens, pool.block_table, 0, 128 ** -0.5)
    torch.testing.assert_close(out.double(), want, rtol=2 ** -7, atol=2 ** -6)   # rounded weights and output, values below 5.5


@pytest.mark.parametrize("variant", ["warp", "tc"])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,page", [(1, 1, 8, 8, 128, 16), (7, 1, 16, 2, 64, 64), (30, 4, 20, 4, 128, 24), (150, 1, 8, 1, 64, 128)])
def test_every_key_counts_once(B, T, Hq, Hkv, D, page, variant):
    """Queries of zero give every key a weight of one, and the log-sum-exp is the logarithm of the number of visible keys, whatever the ranges. Fewer than
    42000 keys, so one key more or less is 2.3e-5 and more; sums of ones are exact, and what is left is the rounding of logarithms below 11 (log2
    below 16) of a range and of their merge, below ten halves of a unit of 2^-20: 5e-6."""
    from triton_distributed_b200 import ops
    k = torch.randn(64, page, Hkv, D, device="cuda").bfloat16()
    v = torch.ones_like(k)
    q = torch.zeros(B * T, Hq, D, device="cuda", dtype=torch.bfloat16)
    for shared in (1, 128, 129, 1000, 5003, 40000):
        for own in (1, 77, 1900):
            g = torch.Generator().manual_seed(shared + own)
            lens = (shared + torch.randint(T, T + own, (B,), generator=g)).int().cuda()
            if B > 1:
                lens[B // 2] = min(shared, 50)                  # ends inside the shared keys
            table = torch.randint(0, 64, (B, -(-(shared + own + T) // page)), generator=g).int().cuda()
            out, lse = ops.shared_prefix_attention(q, k, v, lens, table, shared, 1.0, tokens=T, return_lse=True, variant=variant)
            seen = (lens.double()[:, None] - T + 1 + torch.arange(T, device="cuda")).clamp_min(0).reshape(-1, 1)
            assert bool(((lse.double() - seen.log()).abs() < 1e-5).logical_or((seen == 0) & (lse == float("-inf"))).all()), (shared, own)
            assert torch.equal(out, (seen > 0).to(out.dtype)[..., None].expand_as(out)), (shared, own)
    ops.check_pipeline_status()


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_drafted_tokens_follow_the_target_at_every_place(sampled, dtype):
    """Sampled drafts, and ones that were looked up: the token at each place, among the sequences that got as far, is distributed as the target's row says. A
    frequency among n sequences is off by more than 5 * sqrt(0.25 / n) once in 1.7e6 times; uniform numbers in steps of 2^-24 add less than 1e-6. The
    probabilities are multiples of 1 / 128, which 16 bits hold, so that the rows' sums are exactly one."""
    from triton_distributed_b200 import ops
    B, K, V = 400000, 3, 6
    g = torch.Generator(device="cuda").manual_seed(11)
    def rows(n):
        parts = (torch.softmax(torch.randn(n, V, device="cuda", generator=g) * 1.2, -1) * 120).floor() + 1
        parts[:, 0] += 128 - parts.sum(-1)
        return (parts / 128).to(dtype)

    p, q = rows(K + 1), rows(K)
    if sampled:
        drafts = torch.stack([torch.multinomial(q[i].float(), B, replacement=True, generator=g) for i in range(K)], 1)
    else:
        drafts = p[:K].float().argmax(-1).expand(B, K).contiguous()
    u = torch.rand(B, K + 1, device="cuda", generator=g)
    accepted, tokens = ops.verify_drafts(drafts, p.expand(B, K + 1, V), u, q.expand(B, K, V) if sampled else None)
    for place in range(K + 1):
        got = tokens[accepted >= place, place]
        n = got.numel()
        assert n > 2000
        want = p[place].double()
        freq = torch.bincount(got, minlength=V).double() / n
        assert float((freq - want).abs().max()) < 5 * (0.25 / n) ** 0.5 + 1e-6, (place, freq, want)
