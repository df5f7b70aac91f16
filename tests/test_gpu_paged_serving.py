"""A serving step on device-resident batches: pages and slots (reserve, release), row writes, attention of drafted trees, accepted
paths; each against a plain model of its definition, in whole numbers or 64 bits, and a run of them together.

Tolerances.  A rounding is off by at most half a step, eps / 2 relative (bf16 2^-8, f32 2^-24).  For the attention, with w the exact
weights, A = sum w |v| and Q = max over the seen tokens of scale * sum |q_d k_d|:
  * a score is off by at most Q * e_s: in f32 (D + 8) roundings of 2^-24; on the tensor cores the query enters as a sum of two bf16
    numbers, which leaves 2^-16 of it, products are exact and sums are f32;
  * a weight is then off by 2 * Q * e_s relative (it and the sum), by 2^-21 for the exponential and the f32 sums, and on the
    tensor cores by 2^-8 for its rounding to bf16: O by A times that, and by 2^-8 |O| for its own rounding to bf16;
  * LSE is off by Q * e_s and a few f32 roundings of itself and of the score's magnitude."""
import numpy as np
import pytest
import torch

from tests.gpu_util import ctx, fa

pytestmark = pytest.mark.gpu
THETA = 500000.0


def i32(x):
    return torch.tensor(np.asarray(x, np.int32).reshape(np.shape(x)), device="cuda")


def pages_of(n, page):
    return -(-n // page)


def clean(c):
    c.synchronize()
    assert c.device_status() == 0


# ---- reserve and release ---------------------------------------------------------------------------

def model_reserve(page, pool, most, table, held, ctx_lens, free, f, new, limit, depths=None):
    table, held = table.copy(), held.copy()
    S = len(held)
    offsets, slots, positions, after = np.zeros(S + 1, np.int64), [], [], ctx_lens.copy()
    given, asked, tokens, refused = 0, 0, 0, []
    for s in range(S):
        offsets[s] = min(tokens, limit)
        L, H = int(ctx_lens[s]), int(held[s])
        n = max(int(new[s]), 0)
        tokens += n
        ok = new[s] >= 0 and L >= 0 and H <= most and L <= H * page and L + n <= most * page and tokens <= limit
        need = max(0, pages_of(L + n, page) - H) if ok else 0
        if ok and need and asked + need > f:
            ok = False
        if need:
            if ok:
                for i in range(need):
                    table[s, H + i] = free[f - 1 - (asked + i)]
                held[s] += need
                given += need
            asked += need
        if not ok:
            refused.append(s)
        else:
            after[s] = L + n
        for j in range(n):
            if len(slots) >= limit:
                break
            at = L + j
            slots.append(table[s, at // page] * page + at % page if ok else -1)
            positions.append((L + (j if depths is None else depths[len(positions)])) if ok else 0)
    offsets[S] = min(tokens, limit)
    slots += [-1] * (limit - len(slots))
    positions += [0] * (limit - len(positions))
    return table, held, f - given, offsets, np.array(slots), np.array(positions), after, refused


def random_pool(rng, S, page, ctx_lens, extra_pages, most, spare=0):
    held = np.array([pages_of(n, page) + (int(rng.integers(0, spare + 1)) if spare else 0) for n in ctx_lens], np.int32)
    held = np.minimum(held, most)
    pool = int(held.sum()) + extra_pages
    order = rng.permutation(pool).astype(np.int32)
    table = np.full((S, most), -1, np.int32)
    at = 0
    for s in range(S):
        table[s, :held[s]] = order[at:at + held[s]]
        at += held[s]
    free = np.full(pool, -7, np.int32)
    free[:pool - at] = order[at:]
    return table, held, free, pool - at, pool


def run_reserve(c, page, pool, most, table, held, lens, free, f, new, limit, depths=None, in_place=False):
    S = len(held)
    b = fa.PagedBatch(S, page, pool, most, i32(table), i32(held), i32(lens), i32(free), i32([f]))
    off, slots, pos = i32(np.full(S + 1, 9)), i32(np.full(limit, 9)), i32(np.full(limit, 9))
    outs = {} if in_place else dict(page_counts_out=torch.empty_like(b.page_counts), free_count_out=torch.empty_like(b.free_count))
    after = b.context_lens if in_place else torch.empty_like(b.context_lens)
    c.paged_batch_reserve(b, i32(new), limit, off, slots, pos, depths=None if depths is None else i32(depths), context_lens_out=after, **outs)
    c.synchronize()
    held_out = (b.page_counts if in_place else outs["page_counts_out"]).cpu().numpy()
    f_out = int((b.free_count if in_place else outs["free_count_out"])[0])
    return b.page_tables.cpu().numpy(), held_out, f_out, off.cpu().numpy(), slots.cpu().numpy(), pos.cpu().numpy(), after.cpu().numpy(), b


def same(got, want):
    for name, g, w in zip(("table", "held", "free count", "offsets", "slots", "positions", "lengths"), got, want):
        assert np.array_equal(np.asarray(g), np.asarray(w)), name


@pytest.mark.parametrize("S,page,hi,new_hi,limit_more,in_place", [
    (1, 16, 0, 1, 0, True), (1, 1, 5, 40, 3, False), (7, 16, 100, 20, 0, True), (33, 5, 60, 9, 17, False), (64, 16, 900, 16, 100, True),
    (1025, 16, 50, 3, 0, False), (1025, 16, 50, 30, 5, True), (2500, 7, 40, 12, 0, True), (3, 64, 5000, 9000, 11, False)])
def test_reserve(S, page, hi, new_hi, limit_more, in_place):
    rng = np.random.default_rng(S + page)
    lens = rng.integers(0, hi + 1, S).astype(np.int32)
    new = rng.integers(0, new_hi + 1, S).astype(np.int32)
    new[-1] = new_hi
    most = pages_of(hi + new_hi, page) + 1
    table, held, free, f, pool = random_pool(rng, S, page, lens, S * pages_of(new_hi, page) + S, most, spare=1)
    limit = int(new.sum()) + limit_more
    want = model_reserve(page, pool, most, table, held, lens, free, f, new, limit)
    assert not want[-1]
    c = ctx()
    got = run_reserve(c, page, pool, most, table, held, lens, free, f, new, limit, in_place=in_place)
    clean(c)
    same(got, want)


def test_reserve_depths_set_positions():
    rng = np.random.default_rng(5)
    lens, new = np.array([30, 0, 17], np.int32), np.array([4, 3, 0], np.int32)
    depths = np.array([0, 1, 1, 2, 0, 0, 1])
    table, held, free, f, pool = random_pool(rng, 3, 16, lens, 5, 4)
    want = model_reserve(16, pool, 4, table, held, lens, free, f, new, 7, depths)
    got = run_reserve(ctx(), 16, pool, 4, table, held, lens, free, f, new, 7, depths)
    clean(ctx())
    same(got, want)
    assert got[5].tolist() == [30, 31, 31, 32, 0, 0, 1]


@pytest.mark.parametrize("S", [40, 1500])
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve_where_the_pages_end(S, in_place):
    """Sequences behind the end of the stack get nothing, those that need no page are served."""
    rng = np.random.default_rng(S)
    lens = rng.integers(0, 30, S).astype(np.int32)
    new = rng.integers(0, 12, S).astype(np.int32)
    table, held, free, f, pool = random_pool(rng, S, 4, lens, S // 2, 12)
    want = model_reserve(4, pool, 12, table, held, lens, free, f, new, int(new.sum()))
    assert 0 < len(want[-1]) < S and f > 0
    c = ctx()
    got = run_reserve(c, 4, pool, 12, table, held, lens, free, f, new, int(new.sum()), in_place=in_place)
    assert c.device_status() == 41 and c.device_status() == 0
    same(got, want)


@pytest.mark.parametrize("case", ["negative_new", "negative_len", "more_tokens_than_pages", "table_full", "limit", "huge"])
def test_reserve_leaves_out_sequences_that_make_no_sense(case):
    rng = np.random.default_rng(2)
    lens, new = np.array([10, 20, 30, 5], np.int32), np.array([3, 4, 5, 6], np.int32)
    table, held, free, f, pool = random_pool(rng, 4, 8, lens, 20, 6)
    limit = 18
    if case == "negative_new":
        new[1] = -4
    elif case == "negative_len":
        lens[2] = -1
    elif case == "more_tokens_than_pages":
        lens[0] = 8 * held[0] + 1
    elif case == "table_full":
        new[1] = 29
        limit = 100
    elif case == "limit":
        limit = 9
    else:
        new[0] = new[1] = 2 ** 31 - 1
        limit = 64
    want = model_reserve(8, pool, 6, table, held, lens, free, f, new, limit)
    assert want[-1]
    c = ctx()
    got = run_reserve(c, 8, pool, 6, table, held, lens, free, f, new, limit)
    assert c.device_status() == 31 and c.device_status() == 0
    same(got, want)


def test_reserve_flags_entries_outside_the_pool():
    c = ctx()
    table = np.array([[5, -1, -1], [99, -1, -1]], np.int32)
    got = run_reserve(c, 4, 8, 3, table, np.array([1, 1], np.int32), np.array([2, 2], np.int32), np.array([0, 1, 2, -3, 0, 0, 0, 0], np.int32), 4,
                      np.array([3, 2], np.int32), 5)
    assert c.device_status() == 35
    assert got[4].tolist() == [22, 23, -1, -1, -1]  # sequence 0's new page is -3, sequence 1's old page is 99
    got = run_reserve(c, 4, 8, 3, table[:1], np.array([1], np.int32), np.array([2], np.int32), np.zeros(8, np.int32), 9, np.array([1], np.int32), 1)
    assert c.device_status() == 40 and got[2] == 8 and got[4].tolist() == [22]


def model_release(page, most, table, held, free, f, keep):
    free, out, at = free.copy(), held.copy(), f
    dropped = False
    for s in range(len(held)):
        if keep[s] < 0 or held[s] < 0 or held[s] > most:
            continue
        out[s] = min(held[s], pages_of(int(keep[s]), page))
        for i in range(held[s] - 1, out[s] - 1, -1):
            if at < len(free):
                free[at] = table[s, i]
                at += 1
            else:
                dropped = True
    return free, out, at, dropped


@pytest.mark.parametrize("S,page,hi", [(1, 16, 0), (1, 1, 50), (9, 16, 300), (64, 16, 2000), (1100, 4, 60), (3, 2, 20000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_release(S, page, hi, in_place):
    rng = np.random.default_rng(S * 3 + page)
    lens = rng.integers(0, hi + 1, S).astype(np.int32)
    keep = np.array([rng.choice([0, n, n // 2, n + 100, max(0, n - 5)]) for n in lens], np.int32)
    most = pages_of(hi, page) + 1
    table, held, free, f, pool = random_pool(rng, S, page, lens, 3, most, spare=1)
    want = model_release(page, most, table, held, free, f, keep)
    c = ctx()
    b = fa.PagedBatch(S, page, pool, most, i32(table), i32(held), i32(lens), i32(free), i32([f]))
    ho, fo = (None, None) if in_place else (torch.empty_like(b.page_counts), torch.empty_like(b.free_count))
    c.paged_batch_release(b, i32(keep), ho, fo)
    clean(c)
    assert np.array_equal(b.free_pages.cpu().numpy(), want[0]) and not want[3]
    assert np.array_equal((b.page_counts if in_place else ho).cpu().numpy(), want[1])
    assert int(b.free_count if in_place else fo) == want[2]
    assert np.array_equal(b.page_tables.cpu().numpy(), table)


def test_release_reports_what_makes_no_sense():
    c = ctx()
    table = np.arange(8, dtype=np.int32).reshape(2, 4)
    b = fa.PagedBatch(2, 4, 8, 4, i32(table), i32([2, 3]), i32([8, 12]), i32([4, 5, 6, 7, 0, 0, 0, 0]), i32([5]))
    c.paged_batch_release(b, i32([-1, 0]))
    assert c.device_status() == 31  # sequence 0 keeps its pages
    assert b.page_counts.tolist() == [2, 0] and b.free_count.item() == 8 and b.free_pages.tolist() == [4, 5, 6, 7, 0, 6, 5, 4]
    b = fa.PagedBatch(2, 4, 8, 4, i32(table), i32([2, 3]), i32([8, 12]), i32([4, 5, 6, 7, 0, 0, 0, 0]), i32([5]))
    c.paged_batch_release(b, i32([0, 0]))  # one page more than the pool has room for
    assert c.device_status() == 40
    assert b.page_counts.tolist() == [0, 0] and b.free_count.item() == 8 and b.free_pages.tolist() == [4, 5, 6, 7, 0, 1, 0, 6]


# ---- row writes ------------------------------------------------------------------------------------

def turned64(x, positions, D, theta=THETA):
    """x [n, heads*D] in 64 bits, neighbouring pairs turned by position * theta^(-2j/D)."""
    x = np.asarray(x, np.float64).reshape(len(positions), -1, D // 2, 2)
    a = np.asarray(positions, np.longdouble)[:, None] * np.power(np.longdouble(np.float32(theta)), -2 * np.arange(D // 2, dtype=np.longdouble) / D)
    a = np.fmod(a, 8 * np.arctan(np.longdouble(1))).astype(np.float64)  # 64 bits of a position of 2^31 leave 2^-22 of the angle
    z = (x[..., 0] + 1j * x[..., 1]) * np.exp(1j * a)[:, None, :]
    return np.stack([z.real, z.imag], -1).reshape(len(positions), -1)


def rows_of(gen, n, width, dtype, scale=1.0):
    x = torch.randn(max(n, 1), width, generator=gen) * scale
    return x.to(fa.torch_dtype(dtype))[:n]


@pytest.mark.parametrize("dtype", [fa.F32, fa.BF16])
@pytest.mark.parametrize("tokens,Hkv,D,off", [(1, 1, 2, 0), (3, 8, 128, 0), (5, 2, 6, 0), (700, 3, 64, 0), (41, 5, 80, 0), (129, 8, 128, 1), (5000, 2, 64, 0)])
def test_write(dtype, tokens, Hkv, D, off):
    gen = torch.Generator().manual_seed(tokens + D)
    rng = np.random.default_rng(tokens)
    w, pool = Hkv * D, tokens + 37
    slots = rng.permutation(pool)[:tokens].astype(np.int32)
    positions = rng.integers(0, 200000, tokens).astype(np.int32)
    positions[0] = 2 ** 31 - 1
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]
    td = fa.torch_dtype(dtype)
    ks, vs, k, v = (rows_of(gen, n, w, dtype) for n in (tokens, tokens, pool, pool))
    def place(x):  # a tensor that starts `off` elements into its allocation
        big = torch.empty(x.numel() + off, dtype=td, device="cuda")
        big[off:] = x.reshape(-1).cuda()
        return big[off:].view(x.shape)
    c = ctx()
    for turn in (True, False):
        dk, dv = place(k), place(v)
        c.paged_kv_write(Hkv, D, i32(slots), i32(positions) if turn else None, THETA, place(ks), place(vs), dk, dv)
        clean(c)
        want_k, want_v = k.double().numpy().copy(), v.double().numpy().copy()
        on = slots >= 0
        new = turned64(ks.double().numpy(), positions, D) if turn else ks.double().numpy()
        want_k[slots[on]], want_v[slots[on]] = new[on], vs.double().numpy()[on]
        got = dk.double().cpu().numpy()
        assert np.array_equal(dv.double().cpu().numpy(), want_v)
        if not turn:
            assert np.array_equal(got, want_k)
            continue
        others = np.setdiff1d(np.arange(pool), slots[on])
        assert np.array_equal(got[others], want_k[others])
        # a pair (x, y): cos and sin to 2^-22 (their own error and the angle's 2^-32 of a turn), two products and a sum of 2^-24 each
        pair = np.abs(ks.double().numpy()).reshape(tokens, -1, 2).sum(-1).repeat(2, -1).reshape(tokens, -1)
        size = pair[on] * 2.0 ** -21 + (np.abs(new[on]) * 2.0 ** -8 if dtype == fa.BF16 else 0)
        assert (np.abs(got[slots[on]] - new[on]) <= size).all()


def test_write_leaves_out_slots_behind_the_pool():
    c = ctx()
    k = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    src = torch.ones(3, 64, device="cuda", dtype=torch.bfloat16)
    c.paged_kv_write(1, 64, i32([2, 4, 2 ** 31 - 1]), None, THETA, src, src, k, v)
    assert c.device_status() == 35
    assert k.float().sum(1).tolist() == [0, 0, 64, 0] and v.float().sum(1).tolist() == [0, 0, 64, 0]


# ---- tree attention --------------------------------------------------------------------------------

def random_tree(rng, n):
    """Ancestor sets as rows of truth values, and depths."""
    sees, depth = np.zeros((n, n), bool), np.zeros(n, np.int64)
    for i in range(n):
        if i and rng.random() > 0.1:
            up = int(rng.integers(max(0, i - 5), i))
            sees[i], depth[i] = sees[up], depth[up] + 1
        sees[i, i] = True
    return sees, depth


def pack_masks(masks, words):
    rows = []
    for m in masks:
        bits = np.zeros((len(m), words * 32), bool)
        bits[:, :m.shape[1]] = m
        rows.append(np.packbits(bits, axis=1, bitorder="little").view(np.int32))
    return np.concatenate(rows)


class TreeCase:
    """Random tensors of a batch; `masks` [n, n] per sequence."""

    def __init__(self, seed, dtype, Hq, Hkv, D, page, lens, nodes, masks=None, spare_rows=0, poison=None, scale=1.0, words_more=0):
        rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.dtype, self.Hq, self.Hkv, self.D, self.page, self.lens, self.nodes = dtype, Hq, Hkv, D, page, list(lens), list(nodes)
        S, T = len(lens), sum(nodes)
        trees = [random_tree(rng, n) for n in nodes]
        self.masks = [t[0] for t in trees] if masks is None else masks
        after = np.array(lens) + np.array(nodes)
        self.most = max(pages_of(int(after.max()), page), 1) + 1
        self.table, self.held, _, _, self.pool = random_pool(rng, S, page, after, 3, self.most)
        self.k, self.v = (rows_of(gen, self.pool * page, Hkv * D, dtype) for _ in range(2))
        self.k, self.v = self.k * scale, self.v
        if poison is not None:  # rows that no sequence has a live or drafted token in
            used = np.zeros(self.pool * page, bool)
            for s in range(S):
                at = np.arange(after[s])
                used[self.table[s, at // page] * page + at % page] = True
            self.k[~used], self.v[~used] = poison, poison
        self.offsets = np.cumsum([0] + list(nodes))
        self.q = rows_of(gen, T + spare_rows, Hq * D, dtype)
        self.positions = np.zeros(T + spare_rows, np.int32)
        for s in range(S):
            self.positions[self.offsets[s]:self.offsets[s + 1]] = lens[s] + trees[s][1]
        self.words = pages_of(max(max(nodes), 1), 32) + words_more
        self.T, self.rows = T, T + spare_rows

    def row(self, s, token):
        return self.table[s, token // self.page] * self.page + token % self.page

    def run(self, c, mask="bits", max_nodes=None, max_context=None, cfg=None, status=0, repeat=1, table=None):
        dt = self.dtype
        b = fa.PagedBatch(len(self.lens), self.page, self.pool, self.most, i32(self.table if table is None else table), i32(self.held), i32(self.lens),
                          i32(np.zeros(self.pool, np.int32)), i32([0]))
        packed = None
        if mask == "bits":
            packed = np.zeros((self.rows, self.words), np.int32)
            if self.T:
                packed[:self.T] = pack_masks([m for m in self.masks if len(m)], self.words)
            packed = i32(packed)
        out = c.create_decode_output_buffer(dt, self.rows, self.Hq, self.D)
        out.fill_(0x7b)
        q, k, v = (x.to(fa.torch_dtype(dt)).cuda() for x in (self.q, self.k, self.v))
        for _ in range(repeat):
            c.decode_paged_tree(b, self.Hq, self.Hkv, self.D, max_nodes or max(max(self.nodes), 1),
                                max_context or max(max(a + n for a, n in zip(self.lens, self.nodes)), 1), i32(self.offsets), i32(self.positions),
                                packed, cfg or fa.config(True), THETA, q, k, v, out)
        assert c.device_status() == status
        self.raw = out.cpu()
        o, lse = c.split_decode_output(out, dt, self.rows, self.Hq, self.D)
        return o.double().cpu().numpy(), lse.double().cpu().numpy()

    def exact(self, masks=None, scale=None, drop=()):
        """(O, LSE, A, Q) of the module's docstring in 64 bits."""
        Hq, Hkv, D, G = self.Hq, self.Hkv, self.D, self.Hq // self.Hkv
        c = 1 / np.sqrt(D) if scale is None else scale
        O, LSE, A, Qm = np.zeros((self.T, Hq, D)), np.zeros((self.T, Hq)), np.zeros((self.T, Hq, D)), np.zeros((self.T, Hq))
        k64, v64 = self.k.double().numpy(), self.v.double().numpy()
        for s, (L, n) in enumerate(zip(self.lens, self.nodes)):
            if not n:
                continue
            a, b = self.offsets[s], self.offsets[s + 1]
            at = self.row(s, np.arange(L + n))
            q = turned64(self.q[a:b].double().numpy(), self.positions[a:b], D).reshape(n, Hkv, G, D)
            seen = np.concatenate([np.ones((n, L), bool), (masks or self.masks)[s]], 1)
            for t in drop:
                if t[0] == s:
                    seen[:, t[1]:t[2]] = False
            K, V = k64[at].reshape(-1, Hkv, D), v64[at].reshape(-1, Hkv, D)
            for i in range(n):
                on = seen[i]
                if not on.any():
                    LSE[a + i] = -np.inf
                    continue
                x = np.einsum("hgd,thd->hgt", q[i], K[on]) * c
                top = x.max(-1, keepdims=True)
                w = np.exp(x - top)
                total = w.sum(-1, keepdims=True)
                w = w / total
                O[a + i] = np.einsum("hgt,thd->hgd", w, V[on]).reshape(Hq, D)
                A[a + i] = np.einsum("hgt,thd->hgd", w, np.abs(V[on])).reshape(Hq, D)
                LSE[a + i] = (top + np.log(total)).reshape(Hq)
                Qm[a + i] = (np.einsum("hgd,thd->hgt", np.abs(q[i]), np.abs(K[on])).max(-1) * c).reshape(Hq)
        return O, LSE, A, Qm

    def check(self, got, want):
        o, lse = got[0][:self.T], got[1][:self.T]
        O, LSE, A, Qm = want
        # whichever route a shape takes: bf16 is held to the tensor cores' bounds
        e_s = (self.D + 8) * 2.0 ** -24 + (2.0 ** -16 if self.dtype == fa.BF16 else 0)
        w = (2 * Qm * e_s + 2.0 ** -21)[..., None] + (2.0 ** -8 if self.dtype == fa.BF16 else 0)
        tol = A * w + (np.abs(O) * 2.0 ** -8 if self.dtype == fa.BF16 else 0) + 1e-30
        assert np.isfinite(o).all() and (np.abs(o - O) <= tol).all(), float((np.abs(o - O) - tol).max())
        dead = np.isneginf(LSE)
        assert np.array_equal(dead, np.isneginf(lse)) and (o[dead] == 0).all()
        ltol = Qm * e_s + 2.0 ** -21 * (1 + np.abs(LSE) + Qm)
        assert (np.abs(lse - LSE)[~dead] <= ltol[~dead]).all()


SHAPES = [  # dtype, Hq, Hkv, D, page
    (fa.F32, 4, 2, 64, 16), (fa.F32, 3, 1, 6, 5), (fa.F32, 8, 8, 128, 16), (fa.F32, 10, 2, 80, 1), (fa.BF16, 32, 8, 128, 16), (fa.BF16, 8, 2, 64, 16),
    (fa.BF16, 6, 2, 128, 64), (fa.BF16, 16, 1, 64, 32), (fa.BF16, 5, 5, 128, 48), (fa.BF16, 4, 2, 96, 16), (fa.BF16, 4, 1, 128, 8),
    (fa.BF16, 8, 1, 128, 128)]
LENGTHS = [  # live tokens and drafted tokens of each sequence
    ([0], [1]), ([5], [1]), ([1], [3]), ([700], [8]), ([63, 64, 65, 127, 128, 129], [1, 1, 1, 2, 3, 5]), ([0, 300, 17, 1000], [7, 0, 16, 31]),
    ([500, 40], [64, 33]), ([2500], [1])]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_tree(shape, lengths):
    t = TreeCase(sum(lengths[0]) + shape[3], *shape, *lengths, spare_rows=2, poison=float("nan"))
    got = t.run(ctx())
    t.check(got, t.exact())
    raw = t.raw  # rows behind the last sequence stay as they were
    L = fa.decode_layout(t.dtype, t.rows, t.Hq, t.D)
    size = t.Hq * t.D * (2 if t.dtype == fa.BF16 else 4)
    assert (raw[t.T * size:L.q_bytes] == 0x7b).all() and (raw[L.lse_byte_offset + 4 * t.T * t.Hq:L.combined_bytes] == 0x7b).all()


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4], SHAPES[5], SHAPES[9]], ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_without_a_mask_the_drafts_are_a_chain_or_all_see_one_another(shape, causal):
    lens, nodes = [0, 100, 333], [70, 1, 200]
    masks = [np.tril(np.ones((n, n), bool)) if causal else np.ones((n, n), bool) for n in nodes]
    t = TreeCase(3, *shape, lens, nodes, masks=masks)
    t.check(t.run(ctx(), mask=None, cfg=fa.config(causal)), t.exact())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4], SHAPES[9]], ids=str)
def test_rows_that_see_nothing_and_masks_without_the_own_bit(shape):
    """Mask rows that are empty: only the live tokens count, and without any O = 0 and LSE = -inf."""
    rng = np.random.default_rng(1)
    masks = [rng.random((n, n)) < 0.3 for n in (9, 40, 5)]
    for m in masks:
        m[::3] = False
    t = TreeCase(4, *shape, [0, 0, 77], [9, 40, 5], masks=masks)
    t.check(t.run(ctx()), t.exact())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4], SHAPES[5], SHAPES[9]], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_drafts_have_no_influence_whatever_they_hold(shape, bad):
    """K and V of a drafted token that is not finite: rows that see it are not finite (from V: in the dims that are bad), rows that do
    not see it are what they are without it."""
    t = TreeCase(6, *shape, [50, 200], [20, 40], poison=bad)
    D, G = t.D, t.Hq // t.Hkv
    clean_k, clean_v = t.k.clone(), t.v.clone()
    t.v[t.row(0, 50 + 7), 3] = bad      # head 0, dim 3
    t.v[t.row(1, 200 + 30), D + 1] = bad  # head 1, dim 1
    t.k[t.row(1, 200 + 35), 0] = float("nan")
    o, lse = t.run(ctx())
    t.k, t.v = clean_k, clean_v
    O, LSE, A, Qm = t.exact()
    bad_o, bad_l = np.zeros(O.shape, bool), np.zeros(LSE.shape, bool)
    bad_o[0:20][t.masks[0][:, 7], :G, 3] = True
    bad_o[20:][t.masks[1][:, 30], G:2 * G, 1] = True
    only_v = bad_o.copy()
    bad_o[20:][t.masks[1][:, 35], :G] = True
    bad_l[20:][t.masks[1][:, 35], :G] = True
    assert bad_o.any() and not np.isfinite(o[:t.T][bad_o]).any() and np.isnan(lse[:t.T][bad_l]).all()
    if not np.isnan(bad):
        assert (o[:t.T][only_v & ~np.repeat(bad_l[..., None], D, -1)] == bad).all()
    o[:t.T][bad_o], lse[:t.T][bad_l] = O[bad_o], LSE[bad_l]
    t.check((o, lse), (O, LSE, A, Qm))


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4]], ids=str)
def test_live_tokens_that_are_not_finite_reach_every_row(shape):
    t = TreeCase(8, *shape, [300], [12])
    t.v[t.row(0, 100), 5] = float("nan")
    t.k[t.row(0, 250), t.D] = float("nan")
    o, lse = t.run(ctx())
    G = t.Hq // t.Hkv
    assert np.isnan(o[:, :G, 5]).all() and np.isnan(o[:, G:2 * G]).all() and np.isnan(lse[:, G:2 * G]).all()
    assert np.isfinite(np.delete(o[:, :G], 5, -1)).all() and np.isfinite(lse[:, :G]).all()


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4], SHAPES[5]], ids=str)
def test_scores_far_apart_and_a_scale_of_its_own(shape):
    t = TreeCase(9, *shape, [400, 30], [10, 33], scale=12.0)
    t.check(t.run(ctx(), cfg=fa.config(True, 0.2)), t.exact(scale=np.float64(np.float32(0.2))))


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4], SHAPES[7]], ids=str)
def test_bounds_above_what_there_is_and_two_runs_alike(shape):
    t = TreeCase(10, *shape, [1000, 0, 200], [5, 12, 1])
    c = ctx()
    a = t.run(c, max_nodes=32, max_context=5000)
    first = t.raw.clone()
    t.check(a, t.exact())
    t.check(t.run(c, max_nodes=32, max_context=5000, repeat=3), t.exact())
    assert torch.equal(first, t.raw)


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4]], ids=str)
def test_pages_outside_the_pool_are_left_out_and_flagged(shape):
    t = TreeCase(11, *shape, [200, 90], [6, 4])
    bad = t.table.copy()
    bad[0, 2], bad[0, 5], bad[1, 1] = -1, t.pool, 2 ** 31 - 1
    got = t.run(ctx(), status=35, table=bad)
    p = t.page
    t.check(got, t.exact(drop=[(0, 2 * p, 3 * p), (0, 5 * p, 6 * p), (1, p, 2 * p)]))


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4]], ids=str)
def test_tokens_behind_the_held_pages_or_the_bound_are_left_out_and_flagged(shape):
    t = TreeCase(12, *shape, [60, 90], [6, 4])
    t.held[0] -= 1
    got = t.run(ctx(), status=35)
    t.check(got, t.exact(drop=[(0, int(t.held[0]) * t.page, 66)]))
    t.held[0] += 1
    t.check(t.run(ctx(), status=35, max_context=80), t.exact(drop=[(1, 80, 94)]))


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[4]], ids=str)
def test_sequences_whose_offsets_make_no_sense_are_not_written(shape):
    t = TreeCase(13, *shape, [60, 90, 30], [6, 4, 5])
    want = t.exact()
    c = ctx()
    o, lse = t.run(c, max_nodes=5, status=7)
    L = fa.decode_layout(t.dtype, t.rows, t.Hq, t.D)
    size = t.Hq * t.D * (2 if t.dtype == fa.BF16 else 4)
    assert (t.raw[:6 * size] == 0x7b).all() and (t.raw[L.lse_byte_offset:L.lse_byte_offset + 24 * t.Hq] == 0x7b).all()
    o[:6], lse[:6] = want[0][:6], want[1][:6]
    t.check((o, lse), want)
    t.offsets = np.array([0, 6, 3, 2 ** 31 - 1])
    t.run(c, status=7)
    assert (t.raw[6 * size:L.q_bytes] == 0x7b).all()


# ---- accepted paths --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,Hkv,D,page,S", [(fa.BF16, 8, 128, 16, 5), (fa.F32, 3, 80, 4, 40), (fa.BF16, 1, 6, 3, 7), (fa.F32, 16, 128, 16, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_accept(dtype, Hkv, D, page, S, in_place):
    """Paths that overlap their own sources, none, whole trees, and more than a batch of rows in flight."""
    rng, gen = np.random.default_rng(S), torch.Generator().manual_seed(S)
    lens, nodes = rng.integers(0, 50, S), rng.integers(1, 40, S)
    most = pages_of(90, page)
    table, held, _, _, pool = random_pool(rng, S, page, lens + nodes, 2, most)
    k, v = (rows_of(gen, pool * page, Hkv * D, dtype) for _ in range(2))
    width = int(nodes.max()) + 1
    path, takes = np.full((S, width), -9, np.int32), np.zeros(S, np.int32)
    want_k, want_v = k.clone(), v.clone()
    for s in range(S):
        takes[s] = rng.integers(0, nodes[s] + 1)
        path[s, :takes[s]] = np.sort(rng.choice(nodes[s], takes[s], replace=False))
        row = lambda t: table[s, t // page] * page + t % page  # noqa: E731
        src, dst = row(lens[s] + path[s, :takes[s]]), row(lens[s] + np.arange(takes[s]))
        want_k[dst], want_v[dst] = k[src], v[src]
    b = fa.PagedBatch(S, page, pool, most, i32(table), i32(held), i32(lens), i32(np.zeros(pool)), i32([0]))
    dk, dv = k.cuda(), v.cuda()
    out = None if in_place else torch.zeros(S, dtype=torch.int32, device="cuda")
    c = ctx()
    c.paged_kv_accept(b, Hkv, D, i32(path), i32(takes), out, dk, dv)
    clean(c)
    assert torch.equal(dk.cpu(), want_k) and torch.equal(dv.cpu(), want_v)
    assert np.array_equal((b.context_lens if in_place else out).cpu().numpy(), lens + takes)


@pytest.mark.parametrize("path,take", [([0, 0], 2), ([2, 1], 2), ([-1, 1], 2), ([0, 9], 2), ([0, 1], 3), ([0, 1], -1), ([0, 2 ** 31 - 1], 2)])
def test_accept_leaves_a_bad_path_alone(path, take):
    c = ctx()
    table = np.array([[3, 1, 0], [2, 9, 9]], np.int32)  # the second sequence is fine
    k = torch.arange(4 * 4 * 8, device="cuda", dtype=torch.float32).view(16, 8)
    v, before = k + 1000, k.clone()
    b = fa.PagedBatch(2, 4, 4, 3, i32(table), i32([2, 1]), i32([2, 1]), i32([0, 0, 0, 0]), i32([0]))
    c.paged_kv_accept(b, 1, 8, i32([path, [0, 2]]), i32([take, 2]), None, k, v)
    assert c.device_status() == 7
    assert b.context_lens.tolist() == [2, 3]
    before[2 * 4 + 2] = before[2 * 4 + 3]
    assert torch.equal(k, before) and torch.equal(v, before + 1000)


# ---- a run of them together ------------------------------------------------------------------------

def serving_setup(dtype, S, Hq, Hkv, D, page, max_nodes, seed):
    pool, most = S * 14, 24
    gen = torch.Generator().manual_seed(seed)
    k = torch.full((pool * page, Hkv * D), float("nan"), dtype=fa.torch_dtype(dtype), device="cuda")
    return fa.PagedBatch(S, page, pool, most), gen, k, k.clone()


class Serving:
    """A serving loop as a program writes it: buffers of fixed size, one step = reserve, write, attend, accept, release."""

    def __init__(self, dtype, Hq, Hkv, D, page, S, cap, max_nodes, max_context, c):
        self.dtype, self.Hq, self.Hkv, self.D, self.S, self.cap, self.max_nodes, self.max_context, self.c = dtype, Hq, Hkv, D, S, cap, max_nodes, max_context, c
        self.batch, _, self.k, self.v = serving_setup(dtype, S, Hq, Hkv, D, page, max_nodes, 0)
        z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
        td = fa.torch_dtype(dtype)
        self.new, self.depths, self.offsets, self.slots, self.positions = z(S), z(cap), z(S + 1), z(cap), z(cap)
        self.mask, self.path, self.takes = z(cap, pages_of(max_nodes, 32)), z(S, max_nodes), z(S)
        self.q = torch.zeros(cap, Hq * D, dtype=td, device="cuda")
        self.k_new, self.v_new = (torch.zeros(cap, Hkv * D, dtype=td, device="cuda") for _ in range(2))
        self.out = c.create_decode_output_buffer(dtype, cap, Hq, D)

    def step(self):
        c, b = self.c, self.batch
        c.paged_batch_reserve(b, self.new, self.cap, self.offsets, self.slots, self.positions, depths=self.depths)
        c.paged_kv_write(self.Hkv, self.D, self.slots, self.positions, THETA, self.k_new, self.v_new, self.k, self.v)
        c.decode_paged_tree(b, self.Hq, self.Hkv, self.D, self.max_nodes, self.max_context, self.offsets, self.positions, self.mask, fa.config(True),
                            THETA, self.q, self.k, self.v, self.out)
        c.paged_kv_accept(b, self.Hkv, self.D, self.path, self.takes, None, self.k, self.v)
        c.paged_batch_release(b, b.context_lens)


@pytest.mark.parametrize("dtype,Hq,Hkv,D,graph", [(fa.BF16, 8, 2, 128, False), (fa.BF16, 8, 2, 128, True), (fa.BF16, 4, 4, 64, True), (fa.F32, 4, 2, 64, True)])
def test_a_serving_loop(dtype, Hq, Hkv, D, graph):
    """Steps of a batch, eager or captured once and replayed, against a plain cache of the accepted tokens."""
    S, page, cap, max_nodes = 5, 16, 120, 24
    rng, gen = np.random.default_rng(77), torch.Generator().manual_seed(77)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = fa.Context(0, stream)
        w = Serving(dtype, Hq, Hkv, D, page, S, cap, max_nodes, 300, c)
        td = fa.torch_dtype(dtype)
        kept_k, kept_v = [np.zeros((0, Hkv * D)) for _ in range(S)], [np.zeros((0, Hkv * D)) for _ in range(S)]
        g = None
        for step in range(9):
            nodes = rng.integers(1, max_nodes + 1, S) if step else np.full(S, max_nodes)
            trees = [random_tree(rng, n) for n in nodes]
            T = int(nodes.sum())
            q, kn, vn = rows_of(gen, cap, Hq * D, dtype), rows_of(gen, cap, Hkv * D, dtype), rows_of(gen, cap, Hkv * D, dtype)
            off = np.cumsum([0] + list(nodes))
            depths, mask, path, takes = np.zeros(cap, np.int32), np.zeros((cap, 1), np.int32), np.zeros((S, max_nodes), np.int32), np.zeros(S, np.int32)
            depths[:T] = np.concatenate([t[1] for t in trees])
            mask[:T] = pack_masks([t[0] for t in trees], 1)
            for s in range(S):
                line = np.flatnonzero(trees[s][0][rng.integers(0, nodes[s])])  # a node's ancestors and itself: a path
                takes[s] = len(line)
                path[s, :len(line)] = line
            for to, x in ((w.new, nodes), (w.depths, depths), (w.mask, mask), (w.path, path), (w.takes, takes)):
                to.copy_(torch.from_numpy(np.asarray(x, np.int32)))
            for to, x in ((w.q, q), (w.k_new, kn), (w.v_new, vn)):
                to.copy_(x)
            w.out.fill_(0x7b)
            if not graph or step == 0:
                w.step()
            else:
                if g is None:
                    stream.synchronize()
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=stream):
                        w.step()
                g.replay()
            assert c.device_status() == 0
            o, lse = c.split_decode_output(w.out, dtype, cap, Hq, D)
            o, lse = o.double().cpu().numpy(), lse.double().cpu().numpy()
            # the reference holds the accepted rows as they were written
            t = TreeCase.__new__(TreeCase)
            t.dtype, t.Hq, t.Hkv, t.D, t.page, t.T, t.nodes, t.lens = dtype, Hq, Hkv, D, 1, T, list(nodes), [len(x) for x in kept_k]
            t.masks, t.offsets, t.q = [x[0] for x in trees], off, q
            t.positions = np.concatenate([len(kept_k[s]) + trees[s][1] for s in range(S)])
            rows_k = torch.from_numpy(turned64(kn[:T].double().numpy(), t.positions, D)).to(td).double().numpy()
            rows_v = vn[:T].double().numpy()
            all_k = [np.concatenate([kept_k[s], rows_k[off[s]:off[s + 1]]]) for s in range(S)]
            all_v = [np.concatenate([kept_v[s], rows_v[off[s]:off[s + 1]]]) for s in range(S)]
            starts = np.cumsum([0] + [len(x) for x in all_k])
            t.row = lambda s, at: starts[s] + at
            t.k, t.v = torch.from_numpy(np.concatenate(all_k)), torch.from_numpy(np.concatenate(all_v))
            O, LSE, A, Qm = t.exact()
            # K in the cache may be the neighbouring number where the rotation is rounded: one more step of its type on a score
            t_e = 2.0 ** -7 if dtype == fa.BF16 else 2.0 ** -20
            tol = A * (2 * Qm * (t_e + 2.0 ** -15) + 2.0 ** -7)[..., None] + np.abs(O) * 2.0 ** -7
            assert (np.abs(o[:T] - O) <= tol).all() and (np.abs(lse[:T] - LSE) <= Qm * (t_e + 2.0 ** -15) + 1e-5).all(), step
            assert (w.out[T * Hq * D * td.itemsize:cap * Hq * D * td.itemsize] == 0x7b).all()
            for s in range(S):
                line = path[s, :takes[s]]
                kept_k[s] = np.concatenate([kept_k[s], rows_k[off[s] + line]])
                kept_v[s] = np.concatenate([kept_v[s], rows_v[off[s] + line]])
                if len(kept_k[s]) > 150:  # the sequence ends, another one takes its place
                    kept_k[s], kept_v[s] = kept_k[s][:0], kept_v[s][:0]
                    w.batch.context_lens[s] = 0
            lens = w.batch.context_lens.tolist()
            assert lens == [len(x) for x in kept_k]
            c.paged_batch_release(w.batch, w.batch.context_lens)
            held = sum(pages_of(n, page) for n in lens)
            assert w.batch.page_counts.tolist() == [pages_of(n, page) for n in lens]
            f = int(w.batch.free_count)
            assert f == w.batch.physical_pages - held
            used = [int(x) for s in range(S) for x in w.batch.page_tables[s, :pages_of(lens[s], page)].tolist()]
            assert sorted(used + w.batch.free_pages[:f].tolist()) == list(range(w.batch.physical_pages))
        del g


def test_one_token_a_sequence_is_plain_decode():
    """Against the single-token decode of the same pool: K in its f32-angle rotation, results within both calls' roundings."""
    Hq, Hkv, D, page = 32, 8, 128, 16
    t = TreeCase(21, fa.BF16, Hq, Hkv, D, page, [700, 1, 90, 3000], [1, 1, 1, 1])
    c = ctx()
    o, lse = t.run(c, mask=None)
    n = np.array(t.lens, np.int32) + 1
    out = c.create_decode_output_buffer(fa.BF16, 4, Hq, D)
    table = np.where(t.table < 0, 0, t.table).astype(np.int32)
    c.decode_paged_batched(fa.BF16, 4, Hq, Hkv, D, page, t.pool, t.most, i32(table), i32(n), i32(t.positions), None, n, t.positions, fa.config(True), THETA,
                           t.q.cuda(), t.k.cuda(), t.v.cuda(), out)
    ro, rl = c.split_decode_output(out, fa.BF16, 4, Hq, D)
    O, LSE, A, Qm = t.exact()
    # both calls are within their bounds of the exact value; the older one's angles are off by position * 2^-25 radians as well
    e = 2.0 ** -16 + 136 * 2.0 ** -24 + 3001 * 2.0 ** -25
    tol = A * ((4 * Qm * e + 2.0 ** -20)[..., None] + 2.0 ** -7) + np.abs(O) * 2.0 ** -7
    assert (np.abs(o - ro.double().cpu().numpy()) <= tol).all()
    assert (np.abs(lse - rl.double().cpu().numpy()) <= 2 * Qm * e + 1e-5).all()


# ---- refusals: none of these launches anything -----------------------------------------------------

def refused(kind, call):
    c = ctx()
    before = c.launch_count()
    with pytest.raises(fa.FlatAttentionError) as e:
        call(c)
    assert e.value.kind == kind, (e.value.kind, e.value.detail)
    assert c.launch_count() == before


def test_refusals_of_the_batch_calls():
    b = fa.PagedBatch(2, 4, 8, 3)
    n2, n3, n5 = i32([1, 1]), i32([0, 0, 0]), i32([0] * 5)
    refused("BufferTooSmall", lambda c: c.paged_batch_reserve(b, n2, 6, n3, n5, n5))
    refused("UnsupportedDtype", lambda c: c.paged_batch_reserve(b, n2.long(), 5, n3, n5, n5))
    refused("ZeroDimension", lambda c: c.paged_batch_reserve(b, n2, 0, n3, n5, n5))
    refused("NullPointer", lambda c: c.paged_batch_reserve(b, None, 5, n3, n5, n5))
    refused("NullPointer", lambda c: c.paged_batch_reserve(b, n2, 5, n3, None, n5))
    refused("UnsupportedShape", lambda c: c.paged_batch_release(b, torch.zeros(4, dtype=torch.int32, device="cuda")[::2]))
    refused("UnsupportedShape", lambda c: c.paged_batch_release(b, torch.zeros(2, dtype=torch.int32)))
    b.raw.page_size = 0
    refused("ZeroDimension", lambda c: c.paged_batch_release(b, n2))
    b.raw.page_size = 2 ** 29
    refused("IndexSpaceExceeded", lambda c: c.paged_batch_release(b, n2))
    b.raw.page_size, b.raw.num_seqs = 4, 65536
    refused("DispatchLimit", lambda c: c.paged_batch_release(b, n2))
    b.raw.num_seqs, b.raw.page_counts = 2, b.page_counts.data_ptr() + 1
    refused("MisalignedBuffer", lambda c: c.paged_batch_release(b, n2))


def test_refusals_of_the_row_calls():
    b = fa.PagedBatch(2, 4, 8, 3)
    t = lambda *n, d=torch.bfloat16: torch.zeros(*n, dtype=d, device="cuda")  # noqa: E731
    one = i32([0])
    refused("BufferTooSmall", lambda c: c.paged_kv_write(2, 64, i32([0, 1]), None, THETA, t(1, 128), t(2, 128), t(4, 128), t(4, 128)))
    refused("BufferTooSmall", lambda c: c.paged_kv_write(2, 64, one, None, THETA, t(1, 128), t(1, 128), t(4, 128), t(3, 128)))
    refused("BufferTooSmall", lambda c: c.paged_kv_write(2, 64, i32([0, 1]), one, THETA, t(2, 128), t(2, 128), t(4, 128), t(4, 128)))
    refused("InvalidRotaryHeadDim", lambda c: c.paged_kv_write(2, 7, one, one, THETA, t(1, 14), t(1, 14), t(4, 14), t(4, 14)))
    refused("InvalidRotaryTheta", lambda c: c.paged_kv_write(2, 64, one, one, 0.0, t(1, 128), t(1, 128), t(4, 128), t(4, 128)))
    refused("UnsupportedHeadDim", lambda c: c.paged_kv_write(1, 256, one, one, THETA, t(1, 256), t(1, 256), t(4, 256), t(4, 256)))
    refused("UnsupportedDtype", lambda c: c.paged_kv_write(2, 64, one, None, THETA, t(1, 128), t(1, 128), t(4, 128), t(4, 128, d=torch.float32)))
    refused("UnsupportedDtype", lambda c: c.paged_kv_write(2, 64, one, None, THETA, *(t(n, 128, d=torch.float16) for n in (1, 1, 4, 4))))
    refused("UnsupportedShape", lambda c: c.paged_kv_write(2, 64, one, None, THETA, t(1, 256)[:, ::2], t(1, 128), t(4, 128), t(4, 128)))
    refused("ZeroDimension", lambda c: c.paged_kv_write(0, 64, one, None, THETA, t(1, 128), t(1, 128), t(4, 128), t(4, 128)))
    refused("BufferTooSmall", lambda c: c.paged_kv_accept(b, 2, 64, i32([[0], [0]]), i32([1, 1]), None, t(32, 128), t(31, 128)))
    refused("LengthMismatch", lambda c: c.paged_kv_accept(b, 2, 64, i32([[0]]), i32([1, 1]), None, t(32, 128), t(32, 128)))
    refused("BufferTooSmall", lambda c: c.paged_kv_accept(b, 2, 64, i32([[0], [0]]), one, None, t(32, 128), t(32, 128)))


def test_refusals_of_the_tree_call():
    b = fa.PagedBatch(2, 4, 8, 3)
    cfg = fa.config(True)

    def call(Hq=4, Hkv=2, D=64, max_nodes=3, max_context=9, offsets=i32([0, 1, 3]), positions=i32([0, 0, 0]), mask=i32([[1], [1], [1]]), cfg=cfg, theta=THETA,
             dtype=torch.bfloat16, rows=3, pool=32, out=None):
        t = lambda *n: torch.zeros(*n, dtype=dtype, device="cuda")  # noqa: E731
        return lambda c: c.decode_paged_tree(b, Hq, Hkv, D, max_nodes, max_context, offsets, positions, mask, cfg, theta, t(rows, Hq * D), t(pool, Hkv * D),
                                             t(pool, Hkv * D), torch.zeros(3 * Hq * (2 * D + 4) if out is None else out, dtype=torch.uint8, device="cuda"))

    refused("InvalidHeadGrouping", call(Hq=5))
    refused("ZeroDimension", call(Hkv=0))
    refused("ZeroDimension", call(max_nodes=0))
    refused("ZeroDimension", call(max_context=0))
    refused("InvalidRotaryHeadDim", call(D=63))
    refused("UnsupportedHeadDim", call(D=130))
    refused("InvalidTheta", call(theta=-1.0))
    refused("InvalidScale", call(cfg=fa.config(True, -1.0)))
    refused("LengthMismatch", call(max_nodes=33))
    refused("LengthMismatch", call(mask=i32([[1], [1]])))
    refused("IndexSpaceExceeded", call(max_nodes=70000, mask=None))
    refused("BufferTooSmall", call(rows=2))
    refused("BufferTooSmall", call(pool=31))
    refused("BufferTooSmall", call(out=100))
    refused("BufferTooSmall", call(offsets=i32([0, 1])))
    refused("UnsupportedDtype", call(dtype=torch.float16, out=10000))


def test_the_first_call_of_a_context_is_refused_inside_a_capture():
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = fa.Context(0, stream)
        b = fa.PagedBatch(1, 4, 8, 3)
        keep = i32([0])
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            keep.add_(0)
            with pytest.raises(fa.FlatAttentionError) as e:
                c.paged_batch_release(b, keep)
        assert "before the capture" in e.value.detail
        c.paged_batch_release(b, keep)  # outside it works, and is what a capture needs
        clean(c)
