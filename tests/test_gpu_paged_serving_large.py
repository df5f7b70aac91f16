"""The serving calls where their launches change shape: thousands of sequences, one sequence over the whole device, blocks of rows that
do not divide, and several contexts and streams.  Models, tolerances and helpers are those of test_gpu_paged_serving."""
import numpy as np
import pytest
import torch

from tests.gpu_util import ctx, fa
from tests.test_gpu_paged_serving import (THETA, TreeCase, clean, i32, model_release, model_reserve, pages_of, random_pool, run_reserve, same)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,page,hi,new_hi", [(4096, 16, 60, 9), (4097, 16, 60, 9), (9000, 3, 20, 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve_for_thousands_of_sequences(S, page, hi, new_hi, in_place):
    rng = np.random.default_rng(S)
    lens, new = rng.integers(0, hi + 1, S).astype(np.int32), rng.integers(0, new_hi + 1, S).astype(np.int32)
    most = pages_of(hi + new_hi, page) + 1
    table, held, free, f, pool = random_pool(rng, S, page, lens, S, most, spare=1)
    limit = int(new.sum()) + 7
    want = model_reserve(page, pool, most, table, held, lens, free, f, new, limit)
    c = ctx()
    got = run_reserve(c, page, pool, most, table, held, lens, free, f, new, limit, in_place=in_place)
    same(got, want)
    assert (c.device_status() != 0) == bool(want[-1])


@pytest.mark.parametrize("limit", [700, 2001, 5000])
def test_reserve_where_tokens_and_pages_end(limit):
    """More tokens than max_new_tokens: the sequences behind are refused, and their pages do not count against those before."""
    rng = np.random.default_rng(limit)
    S, page = 1500, 8
    lens, new = rng.integers(0, 50, S).astype(np.int32), rng.integers(0, 6, S).astype(np.int32)
    table, held, free, f, pool = random_pool(rng, S, page, lens, 130, 12)
    want = model_reserve(page, pool, 12, table, held, lens, free, f, new, limit)
    assert want[-1]
    c = ctx()
    got = run_reserve(c, page, pool, 12, table, held, lens, free, f, new, limit, in_place=True)
    same(got, want)
    assert c.device_status() != 0


def test_lengths_that_pass_31_bits_are_refused():
    c = ctx()
    # the first would end at 2^31 + 1, more than a length can say
    b = fa.PagedBatch(2, 2 ** 20, 1000, 4000, page_counts=i32([2048, 1]), context_lens=i32([2 ** 31 - 2, 5]))
    off, slots, pos = i32([9, 9, 9]), i32([9] * 4), i32([9] * 4)
    b.page_tables[1, 0] = 3
    after = torch.empty_like(b.context_lens)
    c.paged_batch_reserve(b, i32([3, 1]), 4, off, slots, pos, context_lens_out=after)
    c.synchronize()
    assert fa.STATUS[c.device_status()] == "InvalidCacheLength"
    assert off.tolist() == [0, 3, 4] and slots.tolist() == [-1, -1, -1, 3 * 2 ** 20 + 5] and after.tolist() == [2 ** 31 - 2, 6]


@pytest.mark.parametrize("S,page,hi", [(4096, 4, 60), (4097, 4, 60), (300, 1, 3000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_release_for_thousands_of_sequences(S, page, hi, in_place):
    rng = np.random.default_rng(S + page)
    lens = rng.integers(0, hi + 1, S).astype(np.int32)
    most = pages_of(hi, page)
    table, held, free, f, pool = random_pool(rng, S, page, lens, 11, most)
    keep = np.where(rng.random(S) < 0.4, 0, rng.integers(0, hi + 1, S)).astype(np.int32)
    want_free, want_held, want_f, _ = model_release(page, most, table, held, free, f, keep)
    c = ctx()
    b = fa.PagedBatch(S, page, pool, most, i32(table), i32(held), i32(lens), i32(free), i32([f]))
    outs = {} if in_place else dict(page_counts_out=torch.empty_like(b.page_counts), free_count_out=torch.empty_like(b.free_count))
    for _ in range(1 if in_place else 3):  # the counter of the blocks is back at its start
        c.paged_batch_release(b, i32(keep), **outs)
    clean(c)
    got = ((b.page_counts if in_place else outs["page_counts_out"]).cpu().numpy(), int((b.free_count if in_place else outs["free_count_out"])[0]), b.free_pages.cpu().numpy())
    for g, w in zip(got, (want_held, want_f, want_free)):
        assert np.array_equal(np.asarray(g), np.asarray(w))


@pytest.mark.parametrize("dtype,Hkv,D,page,steps", [(fa.BF16, 2, 64, 16, 300), (fa.F32, 1, 6, 5, 600)])
def test_accept_paths_longer_than_a_block(dtype, Hkv, D, page, steps):
    rng, gen = np.random.default_rng(steps), torch.Generator().manual_seed(steps)
    S, n = 3, steps + 40
    lens = np.array([0, 37, 5], np.int32)
    most = pages_of(37 + n, page)
    table, held, _, _, pool = random_pool(rng, S, page, lens + n, 2, most)
    width = Hkv * D
    k, v = (torch.randn(pool * page, width, generator=gen).to(fa.torch_dtype(dtype)) for _ in range(2))
    path, takes = np.full((S, steps), -1, np.int32), np.array([steps, 0, steps - 257 if steps > 300 else 257], np.int32)
    for s in range(S):
        path[s, :takes[s]] = np.sort(rng.choice(n, takes[s], replace=False))
    want_k, want_v = k.clone(), v.clone()
    row = lambda s, t: int(table[s, t // page]) * page + t % page  # noqa: E731
    for s in range(S):
        for j in range(takes[s]):
            want_k[row(s, lens[s] + j)] = k[row(s, lens[s] + path[s, j])]
            want_v[row(s, lens[s] + j)] = v[row(s, lens[s] + path[s, j])]
    c = ctx()
    b = fa.PagedBatch(S, page, pool, most, i32(table), i32(held), i32(lens), i32(np.zeros(pool)), i32([0]))
    kd, vd = k.cuda(), v.cuda()
    c.paged_kv_accept(b, Hkv, D, i32(path), i32(takes), None, kd, vd)
    clean(c)
    assert torch.equal(kd.cpu(), want_k) and torch.equal(vd.cpu(), want_v) and b.context_lens.tolist() == (lens + takes).tolist()


# ---- attention -------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,Hq,Hkv,D,page,lens,nodes", [
    (fa.BF16, 4, 1, 128, 16, [20500], [3]),            # one item over the whole device, a tile or two a part
    (fa.BF16, 2, 1, 64, 64, [19000, 7], [1, 2]),
    (fa.BF16, 4, 1, 64, 16, [10000], [40]),            # two blocks of rows, the same
    (fa.F32, 4, 1, 64, 16, [9000], [3]),
    (fa.BF16, 12, 3, 64, 16, [300, 70], [80, 80]),     # three blocks of rows of three heads: an odd number of items
    (fa.BF16, 3, 1, 128, 32, [500, 1, 129], [90, 43, 10]),
    (fa.BF16, 21, 3, 128, 16, [200], [27]),            # blocks that begin inside a drafted token's heads
    (fa.BF16, 5, 1, 64, 16, [64, 65], [30, 60]),
    (fa.BF16, 64, 2, 64, 16, [100], [3]),              # groups of more than four heads, 32 of them
])
def test_items_over_many_parts_and_blocks_that_do_not_divide(dtype, Hq, Hkv, D, page, lens, nodes):
    t = TreeCase(len(lens) + D, dtype, Hq, Hkv, D, page, lens, nodes, spare_rows=1, poison=float("nan"))
    c = ctx()
    got = t.run(c)
    first = t.raw.clone()
    t.check(got, t.exact())
    t.run(c, repeat=2)
    assert torch.equal(first, t.raw)


@pytest.mark.parametrize("Hq,Hkv,n", [(2, 2, 3), (8, 8, 1), (3, 1, 40), (4, 2, 70)])
def test_items_cut_into_parts_of_every_number(Hq, Hkv, n):
    """Sequences of 1 to 40 tiles, alone and with others: parts that end with their item and parts that do not."""
    c = ctx()
    for tiles in [*range(1, 24), 33, 40]:
        for lens in ([64 * tiles - n - 1], [64 * tiles, 64 * (41 - tiles) + 1], [64 * tiles - n, 5, 64 * tiles - n, 64 * tiles - n]):
            lens = [max(x, 0) for x in lens]
            t = TreeCase(tiles, fa.BF16, Hq, Hkv, 64, 64, lens, [n] + [max(1, n - 2)] * (len(lens) - 1))
            t.check(t.run(c), t.exact())


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(fa.BF16, 4, 2, 64), (fa.BF16, 8, 1, 128), (fa.F32, 2, 1, 32)])
@pytest.mark.parametrize("S", [255, 257, 700])
def test_more_sequences_than_a_block_has_threads(dtype, Hq, Hkv, D, S):
    """Most of them without a drafted token, as in a batch that is padded to a fixed size."""
    rng = np.random.default_rng(S)
    nodes = np.where(rng.random(S) < 0.7, 0, rng.integers(1, 5, S))
    nodes[S // 2:S // 2 + 40] = 0
    nodes[-1] = 2
    t = TreeCase(S, dtype, Hq, Hkv, D, 16, rng.integers(0, 90, S).tolist(), nodes.tolist(), spare_rows=3)
    t.check(t.run(ctx()), t.exact())


@pytest.mark.parametrize("dtype", [fa.BF16, fa.F32])
def test_a_batch_without_drafted_tokens_writes_nothing(dtype):
    t = TreeCase(1, dtype, 4, 2, 64, 16, [5, 70], [0, 0], spare_rows=2)
    t.run(ctx())
    assert (t.raw == 0x7b).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_drafts_that_are_not_finite_in_an_item_of_many_parts(bad):
    """A drafted token's V reaches the rows that see it, whichever CTA has its tile, and no others."""
    Hq, Hkv, D, n = 4, 1, 64, 70
    masks = [np.eye(n, dtype=bool)]
    t = TreeCase(5, fa.BF16, Hq, Hkv, D, 16, [6000], [n], masks=masks)
    want = t.exact()
    at = t.row(0, 6000 + 66)
    t.v[at, 9] = bad
    o, lse = t.run(ctx())
    assert (np.isnan(o[66, :, 9]) if bad != bad else np.isinf(o[66, :, 9])).all()
    o[66, :, 9] = want[0][66, :, 9]
    t.check((o, lse), want)


def test_contexts_and_streams_have_nothing_in_common():
    """Two contexts, each on a stream of its own, called in turn without a wait between them; then one moved to the other stream."""
    cases = [TreeCase(31, fa.BF16, 8, 2, 128, 16, [900, 40], [9, 3]), TreeCase(32, fa.BF16, 8, 2, 128, 16, [100, 2000], [16, 7])]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    contexts, calls, outs = [], [], []
    for t, stream in zip(cases, streams):
        with torch.cuda.stream(stream):
            c = fa.Context(0, stream)
            b = fa.PagedBatch(len(t.lens), t.page, t.pool, t.most, i32(t.table), i32(t.held), i32(t.lens), i32(np.zeros(t.pool)), i32([0]))
            packed = np.zeros((t.rows, t.words), np.int32)
            for s, m in enumerate(t.masks):
                for i in range(len(m)):
                    packed[t.offsets[s] + i, 0] = sum(1 << int(j) for j in np.flatnonzero(m[i]))
            out = c.create_decode_output_buffer(fa.BF16, t.rows, t.Hq, t.D)
            args = (b, t.Hq, t.Hkv, t.D, max(t.nodes), max(t.lens) + max(t.nodes), i32(t.offsets), i32(t.positions), i32(packed), fa.config(True), THETA,
                    t.q.cuda(), t.k.cuda(), t.v.cuda(), out)
        contexts.append(c)
        calls.append(args)
        outs.append(out)
    torch.cuda.synchronize()
    for _ in range(20):
        for c, args in zip(contexts, calls):
            c.decode_paged_tree(*args)
    torch.cuda.synchronize()
    contexts[0].set_stream(streams[1])
    for _ in range(3):
        contexts[0].decode_paged_tree(*calls[0])
    for t, c, out in zip(cases, contexts, outs):
        assert c.device_status() == 0
        o, lse = c.split_decode_output(out, fa.BF16, t.rows, t.Hq, t.D)
        t.check((o.double().cpu().numpy(), lse.double().cpu().numpy()), t.exact())


def test_a_captured_call_follows_the_lengths_on_the_device():
    """One capture, replayed over batches whose lengths, tables and trees change under it."""
    Hq, Hkv, D, page, S, most, nodes_max = 8, 2, 64, 16, 4, 40, 12
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = fa.Context(0, stream)
        rng = np.random.default_rng(3)
        pool, rows = S * most, S * nodes_max
        t = lambda *n: torch.zeros(*n, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        b = fa.PagedBatch(S, page, pool, most)
        off, pos, mask = i32(np.zeros(S + 1)), i32(np.zeros(rows)), i32(np.zeros((rows, 1)))
        q, k, v = t(rows, Hq * D), t(pool * page, Hkv * D), t(pool * page, Hkv * D)
        out = c.create_decode_output_buffer(fa.BF16, rows, Hq, D)
        call = lambda: c.decode_paged_tree(b, Hq, Hkv, D, nodes_max, most * page, off, pos, mask, fa.config(True), THETA, q, k, v, out)  # noqa: E731
        call()
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call()
        for step in range(4):
            lens, nodes = rng.integers(0, 600, S).tolist(), rng.integers(0, nodes_max + 1, S).tolist()
            nodes[step] = nodes_max
            x = TreeCase(100 + step, fa.BF16, Hq, Hkv, D, page, lens, nodes, spare_rows=rows - sum(nodes))
            table = np.zeros((S, most), np.int32)
            table[:, :x.table.shape[1]] = x.table
            packed = np.zeros((rows, 1), np.int32)
            for s, m in enumerate(x.masks):
                for i in range(len(m)):
                    packed[x.offsets[s] + i, 0] = sum(1 << int(j) for j in np.flatnonzero(m[i]))
            for to, src in ((b.page_tables, table), (b.page_counts, x.held), (b.context_lens, lens), (off, x.offsets), (pos, x.positions), (mask, packed)):
                to.copy_(torch.from_numpy(np.asarray(src, np.int32)))
            q.copy_(x.q)
            k[:x.pool * page].copy_(x.k)
            v[:x.pool * page].copy_(x.v)
            out.fill_(0x7b)
            g.replay()
            assert c.device_status() == 0
            o, lse = c.split_decode_output(out, fa.BF16, rows, Hq, D)
            x.check((o.double().cpu().numpy(), lse.double().cpu().numpy()), x.exact())
        del g


@pytest.mark.parametrize("dtype", [fa.BF16, fa.F32])
def test_a_pool_of_more_than_2_to_the_31_elements(dtype):
    """The same rows at the pool's beginning and behind its 2^31-th element (byte offsets behind 2^32): written, attended and moved alike."""
    Hq, Hkv, D, page = 16, 8, 128, 16
    td = fa.torch_dtype(dtype)
    pool = (2 ** 31 // (Hkv * D) + 4096) // page
    k, v = (torch.empty(pool * page, Hkv * D, dtype=td, device="cuda") for _ in range(2))
    t = TreeCase(41, dtype, Hq, Hkv, D, page, [300, 45], [9, 20])
    c = ctx()
    results = []
    for at in (0, pool - t.pool):
        rows = slice(at * page, (at + t.pool) * page)
        k[rows], v[rows] = t.k.to(td).cuda(), t.v.to(td).cuda()
        b = fa.PagedBatch(2, page, pool, t.most, i32(np.where(t.table < 0, -1, t.table + at)), i32(t.held), i32(t.lens), i32(np.zeros(pool)), i32([0]))
        slots = i32(np.concatenate([t.row(s, np.arange(a, a + n)) for s, (a, n) in enumerate(zip(t.lens, t.nodes))]) + at * page)
        new = [torch.randn(t.T, Hkv * D, generator=torch.Generator().manual_seed(7)).to(td).cuda() for _ in range(2)]
        c.paged_kv_write(Hkv, D, slots, i32(t.positions), THETA, new[0], new[1], k, v)
        out = c.create_decode_output_buffer(dtype, t.rows, Hq, D)
        out.fill_(0)
        c.decode_paged_tree(b, Hq, Hkv, D, 20, 400, i32(t.offsets), i32(t.positions), None, fa.config(True), THETA, t.q.to(td).cuda(), k, v, out)
        c.paged_kv_accept(b, Hkv, D, i32([[0, 2, 7], [5, 19, -1]]), i32([3, 2]), None, k, v)
        clean(c)
        results.append((out.cpu(), k[rows].cpu(), v[rows].cpu(), b.context_lens.cpu()))
    for x, y in zip(*results):
        assert torch.equal(x, y)
    assert not torch.equal(results[0][1], t.k.to(td)) and results[0][3].tolist() == [303, 47]


def test_refusals_of_more_rows_than_a_launch_takes():
    b = fa.PagedBatch(1, 16, 4, 4)
    t = lambda n: torch.zeros(n, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    c = ctx()
    before = c.launch_count()
    with pytest.raises(fa.FlatAttentionError) as e:
        c.decode_paged_tree(b, 512, 1, 2, 65535, 60, i32([0, 1]), i32([0]), None, fa.config(True), THETA, t(1024), t(128), t(128), torch.zeros(8192, dtype=torch.uint8, device="cuda"))
    assert e.value.kind == "DispatchLimit" and c.launch_count() == before
