"""The serving calls at the limits of what a batch may hold: tokens cut off by a bound or by the pages held, infinite K in tokens
that are seen, faults reported next to one another, results that take the place of a batch's tensors.  Models, tolerances and helpers are those of test_gpu_paged_serving."""
import numpy as np
import pytest
import torch

from tests.gpu_util import ctx, fa
from tests.test_gpu_decode_cache import _one_sequence_slice
from tests.test_gpu_paged_serving import THETA, TreeCase, clean, i32, turned64

pytestmark = pytest.mark.gpu


# ---- tokens that a bound or the pages held cut off, inside a tile that holds live tokens only -------

CLIPPED = [  # live tokens, drafted tokens, and the tokens that are left of each sequence: by max_context, or by the pages held
    ([140], [5], 80, None), ([140], [5], 70, None), ([140], [5], None, [6]), ([140], [5], None, [0]), ([140], [70], 80, None), ([140], [70], None, [5]),
    ([150, 1000, 30], [5, 3, 2], 500, None), ([150, 1000, 30], [40, 33, 2], 500, None), ([700, 200, 90], [3, 70, 1], None, [20, 1, 0]),
    ([6000], [3], 4010, None), ([6000], [40], 4010, None), ([9000, 700], [2, 5], None, [301, 2])]


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(fa.BF16, 4, 1, 64), (fa.BF16, 8, 2, 128), (fa.F32, 4, 2, 64)])
@pytest.mark.parametrize("lens,nodes,most,held", CLIPPED, ids=str)
def test_live_tokens_that_are_cut_off_do_not_count(dtype, Hq, Hkv, D, lens, nodes, most, held):
    """Products of 64 and of 128 rows, items of one CTA and of many parts."""
    t = TreeCase(sum(lens) + D, dtype, Hq, Hkv, D, 16, lens, nodes)
    left = [most] * len(lens)
    if held is not None:
        left = [n * t.page for n in held]
        t.held = np.array(held, np.int32)
    got = t.run(ctx(), max_context=most, status=35)
    t.check(got, t.exact(drop=[(s, n, a + b) for s, (n, a, b) in enumerate(zip(left, lens, nodes)) if n < a + b]))


# ---- K that is infinite in a token that is seen ------------------------------------------------------

@pytest.mark.parametrize("shape", [(fa.BF16, 8, 2, 128, 16), (fa.BF16, 8, 2, 64, 16), (fa.BF16, 4, 2, 96, 16), (fa.F32, 4, 2, 64, 16)], ids=str)
@pytest.mark.parametrize("lens,nodes", [([90], [9]), ([300, 20], [40, 3]), ([5000], [3])], ids=str)
@pytest.mark.parametrize("exact_queries", [False, True])
def test_an_infinite_k_counts_for_nothing_where_the_score_falls_and_makes_the_row_nan_where_it_rises(shape, lens, nodes, exact_queries):
    """Products with an infinity have the query's sign: a score of -inf has weight 0, one of +inf leaves no weights.  exact_queries:
    turned and scaled queries that are bf16 numbers, of which nothing is left over for a second summand."""
    t = TreeCase(sum(lens) + shape[3], *shape, lens, nodes)
    cfg, scale = fa.config(True), None
    if exact_queries:
        f = np.float32
        scale = next(x for x in (f(1) / f(1.4426950408889634) + f(i) * f(2.0 ** -24) for i in (0, 1, -1, 2, -2)) if f(x) * f(1.4426950408889634) == f(1))
        cfg, scale = fa.config(True, float(scale)), float(scale)
        t.positions[:] = 0
    D, G = t.D, t.Hq // t.Hkv
    at = t.row(0, lens[0] // 2)
    want = t.exact(scale=scale, drop=[(0, lens[0] // 2, lens[0] // 2 + 1)])
    q = turned64(t.q[:t.T].double().numpy(), t.positions[:t.T], D).reshape(t.T, t.Hq, D)[:nodes[0]]
    t.k[at, 6], t.k[at, D + 7] = float("inf"), -float("inf")  # head 0, dim 6; head 1, dim 7
    signs = np.concatenate([q[:, :G, 6], -q[:, G:2 * G, 7]], 1)
    assert (np.abs(signs) > 2.0 ** -20).all() and (signs < 0).any() and (signs > 0).any()
    o, lse = t.run(ctx(), cfg=cfg)
    rises = np.zeros((t.T, t.Hq), bool)
    rises[:nodes[0], :2 * G] = signs > 0
    assert np.isnan(o[rises]).all() and np.isnan(lse[rises]).all()
    o[rises], lse[rises] = want[0][rises], want[1][rises]
    t.check((o, lse), want)


# ---- faults reported next to one another -------------------------------------------------------------

def write_behind_the_pool(c, bad, tokens=2000):
    """A row write whose tokens `bad` name slots behind the pool."""
    src, pool = torch.ones(tokens, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(tokens, 64, device="cuda", dtype=torch.bfloat16)
    slots = np.arange(tokens)
    slots[bad] = tokens + 5
    c.paged_kv_write(1, 64, i32(slots), None, THETA, src, src, pool, pool.clone())


def test_a_wait_that_gave_up_is_not_hidden_by_what_is_reported_behind_it():
    """The exchange waits for a rank that does not exist and gives up after about a second (a bounded wait); a bad slot is reported
    behind it, before the status is read.  What gave up may have left counters half way: the status has to say so."""
    c = fa.Context(0)
    t = TreeCase(55, fa.BF16, 8, 2, 128, 16, [900, 40], [9, 3])
    want = t.exact()
    t.check(t.run(c), want)
    args, Hq, D = _one_sequence_slice(16 * 40)
    x = fa.SplitKvPeerExchange(c, 0, 2, Hq, D)
    try:
        x.connect(x.handle() * 2)
        out = c.create_decode_output_buffer(fa.BF16, 1, Hq, D)
        c.splitkv_decode_peer(x, fa.BF16, *args, out)
        write_behind_the_pool(c, [3])
        c.synchronize()
        assert fa.STATUS[c.device_status()] == "DeviceWaitTimeout"
        assert c.device_status() == 0
    finally:
        x.close()
    t.check(t.run(c), want)
    clean(c)
    c.close()


def test_what_the_status_names_does_not_depend_on_the_order_of_the_blocks():
    c = ctx()
    for _ in range(20):
        write_behind_the_pool(c, [3, 700, 1400, 1999])
        assert c.device_status() == 35
        assert "1999" in fa.lib().flat_last_error_detail(c.h).decode()


def told(c, kind):
    """What the status says, once: its words."""
    assert fa.STATUS[c.device_status()] == kind
    text = fa.lib().flat_last_error_detail(c.h).decode()
    assert c.device_status() == 0
    return text


@pytest.mark.parametrize("shape", [(fa.F32, 4, 2, 64, 16), (fa.BF16, 8, 2, 128, 16)], ids=str)
def test_the_words_of_a_fault_of_the_attention_name_what_was_met(shape):
    c = ctx()
    t = TreeCase(12, *shape, [60, 90], [6, 4])
    t.run(c, max_context=80, status=35)
    assert "sequence 1 has more tokens than its pages or max_context hold" in fa.lib().flat_last_error_detail(c.h).decode()
    t.held[0] -= 1
    t.run(c, status=35)
    assert "sequence 0 has more tokens" in fa.lib().flat_last_error_detail(c.h).decode()
    t.held[0] += 1
    bad = t.table.copy()
    bad[1, 2] = t.pool
    t.run(c, table=bad, status=35)
    assert "a page-table entry of sequence 1 lies outside the physical pool" in fa.lib().flat_last_error_detail(c.h).decode()
    t.run(c, max_nodes=5, status=7)
    assert "lengths of sequence 0 do not fit" in fa.lib().flat_last_error_detail(c.h).decode()


def test_the_words_of_a_fault_of_the_other_calls_name_what_was_met():
    c = ctx()
    write_behind_the_pool(c, [7])
    assert "the slot of token 7 lies behind the pool" in told(c, "PageOutOfRange")
    src, pool = torch.ones(3, 6, device="cuda"), torch.zeros(8, 6, device="cuda")  # rows that are not whole vectors
    c.paged_kv_write(1, 6, i32([1, 9, 2]), None, THETA, src, src, pool, pool.clone())
    assert "the slot of token 1 lies behind the pool" in told(c, "PageOutOfRange")
    k = torch.zeros(32, 8, device="cuda")
    b = fa.PagedBatch(2, 4, 8, 3, i32([[3, 1, 0], [2, 4, 9]]), i32([2, 2]), i32([2, 1]))
    c.paged_kv_accept(b, 1, 8, i32([[0, 1], [1, 1]]), i32([2, 2]), None, k, k.clone())
    assert "the accepted path of sequence 1 does not rise" in told(c, "LengthMismatch")
    b = fa.PagedBatch(2, 4, 8, 3, i32([[3, 1, 0], [2, 99, 9]]), i32([1, 2]), i32([2, 1]), i32([0, 4, 5, 6, 7, 0, 0, 0]), i32([5]))
    c.paged_batch_release(b, i32([4, 0]))
    assert "a page of sequence 1 lies outside the physical pool" in told(c, "PageOutOfRange")
    b = fa.PagedBatch(2, 4, 8, 3, i32([[3, 1, 0], [2, 4, 9]]), i32([2, 2]), i32([2, 1]), i32([0] * 8), i32([8]))
    c.paged_batch_release(b, i32([8, 0]))
    assert "no room for the pages that sequence 1 gives back" in told(c, "CapacityOverflow")
    b.free_count = i32([9])
    c.paged_batch_release(b, i32([8, 0]))
    assert "the count of free pages lies outside the pool" in told(c, "CapacityOverflow")
    b = fa.PagedBatch(2, 4, 8, 3, i32([[3, 1, 0], [2, 4, 9]]), i32([2, 2]), i32([2, 1]), i32([0] * 8), i32([0]))
    c.paged_batch_reserve(b, i32([0, 9]), 9, i32([0] * 3), i32([0] * 9), i32([0] * 9))
    assert "the free pages do not hold the new tokens of sequence 1" in told(c, "CapacityExceeded")


# ---- results of a call out of place that take the place of the batch's tensors -----------------------

def test_counts_written_out_of_place_are_used_once_they_are_the_batch_s():
    c = ctx()
    new, keep = i32([5, 0, 17]), i32([3, 0, 20])
    batches = [fa.PagedBatch(3, 4, 20, 8) for _ in range(2)]
    rows = [[torch.zeros(n, dtype=torch.int32, device="cuda") for n in (4, 22, 22)] for _ in batches]
    for step in range(2):
        a, b = batches
        c.paged_batch_reserve(a, new, 22, *rows[0], context_lens_out=a.context_lens)
        counts, free, lens = torch.empty_like(b.page_counts), torch.empty_like(b.free_count), torch.empty_like(b.context_lens)
        c.paged_batch_reserve(b, new, 22, *rows[1], page_counts_out=counts, free_count_out=free, context_lens_out=lens)
        b.page_counts, b.free_count, b.context_lens = counts, free, lens
        for x, y in zip(*rows):
            assert torch.equal(x, y), step
        c.paged_batch_release(a, keep)
        counts, free = torch.empty_like(b.page_counts), torch.empty_like(b.free_count)
        c.paged_batch_release(b, keep, counts, free)
        b.page_counts, b.free_count = counts, free
        for batch in batches:
            batch.context_lens = keep.clone()
        assert c.device_status() == (31 if step else 0)  # 20 + 17 tokens are more than the 8 pages of a row of the table
        assert a.page_counts.tolist() == b.page_counts.tolist() == [1, 0, 5] and a.free_count.item() == b.free_count.item() == 14
        assert torch.equal(a.free_pages[:14], b.free_pages[:14])
