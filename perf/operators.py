"""The measured operators of speculative serving over a paged K/V pool: page tables and slot maps made on the device, the
write of new rows through a slot map, attention of drafted token trees, and the move of the accepted rows.

A pool holds `pages` pages of `page` tokens, a row of kv_heads * head_dim values a token.  A sequence has `ctx` live tokens and
holds the pages that they need; a step adds `new` (drafted) tokens behind them.  Lengths that vary inside a batch come from the
case itself (`lengths`), so that a case always means the same sizes; what the tensors hold comes from the seed.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False
THETA = 500000.0
_kept = {}


def framework():
    """The package of this repository (its folder name is not a Python identifier)."""
    if "fa" not in _kept:
        _kept["fa"] = importlib.import_module("flat-attention_b200")
    return _kept["fa"]


def context():
    """One context for the process, as a program keeps it."""
    if "ctx" not in _kept:
        _kept["ctx"] = framework().Context(0)
    return _kept["ctx"]


# ---- the cases -----------------------------------------------------------------------------------

def listed():
    return [
        # the step of a full speculative batch: 64 sequences, a small tree each, hardly any page to take
        dict(name="reserve_step", op="reserve", S=64, lo=512, hi=8192, new_lo=1, new_hi=16, page=16, lengths=3),
        # admission of many prompts at once: every page and every slot is new
        dict(name="reserve_prompts", op="reserve", S=2048, lo=0, hi=200, new_lo=1, new_hi=1024, page=16, lengths=4),
        # the end of a step: some sequences finish, others give back what their rejected drafts took
        dict(name="release_step", op="release", S=64, lo=512, hi=8192, page=16, lengths=5),
        # a batch of an evaluation ends, or a node is drained
        dict(name="release_many", op="release", S=4096, lo=512, hi=8192, page=16, lengths=6),
        # drafted trees of a batch enter the cache
        dict(name="write_step", op="write", dtype="bf16", S=64, lo=512, hi=8192, new_lo=1, new_hi=16, Hkv=8, D=128, page=16, lengths=7),
        # prompt chunks of 2048 tokens of several sequences enter the cache
        dict(name="write_chunks", op="write", dtype="bf16", S=16, lo=0, hi=30000, new_lo=2048, new_hi=2048, Hkv=8, D=128, page=16, lengths=8),
        # the accepted paths of a batch
        dict(name="accept_step", op="accept", dtype="bf16", S=64, lo=100, hi=1000, new_lo=8, new_hi=16, take=5, Hkv=8, D=128, page=16, lengths=9),
        # large trees, long paths, many sequences
        dict(name="accept_many", op="accept", dtype="bf16", S=512, lo=0, hi=300, new_lo=33, new_hi=64, take=16, Hkv=8, D=128, page=16, lengths=10),
        # one interactive user with a tree of eight nodes: latency
        dict(name="tree_one", op="tree", dtype="bf16", S=1, lo=700, hi=700, new_lo=8, new_hi=8, Hq=32, Hkv=8, D=128, page=16, lengths=1),
        # the f32 mode of a small model
        dict(name="tree_f32", op="tree", dtype="f32", S=3, lo=33, hi=1500, new_lo=5, new_hi=13, Hq=8, Hkv=2, D=64, page=16, lengths=11),
        # an ordinary serving batch with trees of up to 16 nodes
        dict(name="tree_batch", op="tree", dtype="bf16", S=32, lo=512, hi=8192, new_lo=4, new_hi=16, Hq=32, Hkv=8, D=128, page=16, lengths=12),
        # the largest: a full batch with large trees
        dict(name="tree_wide", op="tree", dtype="bf16", S=64, lo=512, hi=8192, new_lo=33, new_hi=64, Hq=32, Hkv=8, D=128, page=16, lengths=5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    c = dict(op=rng.choice(["reserve", "release", "write", "accept", "tree", "tree"]), page=rng.choice([16, 16, 32, 64]), lengths=rng.randrange(1 << 20))
    if c["op"] == "reserve":
        c["S"] = _log_int(rng, 1, 2048)
        c["new_lo"], c["new_hi"] = 0, _log_int(rng, 1, 1000)
        c["lo"], c["hi"] = 0, _log_int(rng, 1, 400000 // c["S"])
        return c
    if c["op"] == "release":
        c["S"] = _log_int(rng, 1, 4000)
        c["lo"], c["hi"] = 0, _log_int(rng, 1, 8000)
        return c
    c["dtype"] = rng.choice(["bf16", "bf16", "bf16", "f32"])
    c["Hkv"], c["D"] = rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 128]) if c["dtype"] == "bf16" else rng.choice([32, 64, 80, 128])
    if c["op"] == "write":
        c["S"], c["new_lo"], c["new_hi"] = _log_int(rng, 1, 64), 0, _log_int(rng, 1, 400 if c["dtype"] == "bf16" else 200)
        c["lo"], c["hi"] = 0, _log_int(rng, 100, 100000)
        return c
    if c["op"] == "accept":
        c["S"], c["new_lo"], c["new_hi"] = _log_int(rng, 1, 400 if c["dtype"] == "bf16" else 200), 1, _log_int(rng, 2, 64)
        c["take"], c["lo"], c["hi"] = rng.randint(1, 16), 0, _log_int(rng, 10, 300)
        return c
    c["Hq"] = c["Hkv"] * rng.choice([1, 2, 3, 4, 4, 8] if c["Hkv"] < 8 else [1, 2, 4])
    most = 250000 if c["dtype"] == "bf16" else 8000  # tokens of the batch
    c["S"] = _log_int(rng, 1, 64 if c["dtype"] == "bf16" else 8)
    c["new_lo"], c["new_hi"] = 1, _log_int(rng, 1, 64 if c["dtype"] == "bf16" else 24)
    c["hi"] = _log_int(rng, 20, min(16000 if c["S"] == 1 else 8000, most // c["S"]))
    c["lo"] = rng.choice([0, c["hi"] // 16])
    return c


def _lengths(case):
    """(live tokens, new tokens or tokens to keep) of each sequence."""
    rng = random.Random(case["lengths"])
    ctx = [rng.randint(case["lo"], case["hi"]) for _ in range(case["S"])]
    if case["op"] == "release":
        return ctx, [rng.choice([0, n, max(0, n - rng.randint(1, 40)), n // 2]) for n in ctx]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["S"])]
    return ctx, new if sum(new) else [1] * case["S"]


def _takes(case, new):
    """Accepted tokens of each sequence."""
    rng = random.Random(case["lengths"] + 1)
    return [rng.randint(0, min(case["take"], n)) for n in new]


def _pages(n, page):
    return -(-n // page)


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


# ---- what a program has in hand ------------------------------------------------------------------

def _trees(rng, new):
    """Packed (depth, parents, ancestor sets as integers with the node's own bit) of one random tree a sequence; now and then a
    node starts a tree of its own."""
    depth, sees = [], []
    for n in new:
        d, a = [], []
        for i in range(n):
            up = -1 if i == 0 or rng.random() < 0.03 else rng.randrange(max(0, i - 6), i)
            d.append(0 if up < 0 else d[up] + 1)
            a.append((1 << i) | (0 if up < 0 else a[up]))
        depth += d
        sees += a
    return depth, sees


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ctx, new = _lengths(case)
    S, page, op = case["S"], case["page"], case["op"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    after = ctx if op == "release" else [a + b for a, b in zip(ctx, new)]
    held = [_pages(n, page) for n in ctx]
    most = max(max(_pages(n, page) for n in after), 1)
    mapped = held if op in ("reserve", "release") else [_pages(n, page) for n in after]  # pages that the table names
    pool = sum(_pages(n, page) for n in after) + max(4, S // 4)
    order = rng.permutation(pool).astype(np.int32)
    table = np.full((S, most), -1, np.int32)
    ends = np.cumsum([0] + mapped)
    table[np.arange(most)[None, :] < np.array(mapped)[:, None]] = order[:ends[-1]]
    free = np.zeros(pool, np.int32)
    free[:pool - ends[-1]] = order[ends[-1]:]
    st = dict(case=case, op=op, table=torch.from_numpy(table).cuda(), free=torch.from_numpy(free).cuda(), free_count=i32([pool - int(ends[-1])]),
              held=i32(mapped), ctx=i32(ctx), new=i32(new), pool=pool, most=most)
    tokens = sum(new)
    if op in ("reserve", "release"):
        st.update(tokens=tokens, held_out=torch.zeros_like(st["held"]), free_count_out=torch.zeros_like(st["free_count"]),
                  offsets=torch.zeros(S + 1, dtype=torch.int32, device="cuda"), slots=torch.zeros(max(tokens, 1), dtype=torch.int32, device="cuda"),
                  positions=torch.zeros(max(tokens, 1), dtype=torch.int32, device="cuda"))
    else:
        dt, Hkv, D = _type(case), case["Hkv"], case["D"]
        rows = lambda n, w: torch.randn(n, w, generator=gen, device="cuda", dtype=dt)  # noqa: E731
        st["k"], st["v"] = rows(pool * page, Hkv * D), rows(pool * page, Hkv * D)
        seq = np.repeat(np.arange(S), new)
        j = np.arange(tokens) - np.repeat(np.cumsum([0] + new)[:-1], new)
        at = np.array(ctx)[seq] + j
        if op == "write":
            st["slots"] = i32(table[seq, at // page].astype(np.int64) * page + at % page)
            st["positions"] = i32(at)
            st["k_new"], st["v_new"] = rows(tokens, Hkv * D), rows(tokens, Hkv * D)
        elif op == "accept":
            takes = _takes(case, new)
            width = max(max(takes), 1)
            path = np.full((S, width), -1, np.int32)
            for s, (n, a) in enumerate(zip(new, takes)):  # the likeliest chain comes first; the path leaves it for a later node
                c = int(rng.integers(max(0, 2 * a - n), a + 1))
                path[s, :a] = list(range(c)) + sorted(rng.choice(np.arange(a, n), a - c, replace=False).tolist())
            st.update(path=torch.from_numpy(path).cuda(), takes=i32(takes), ctx_out=torch.zeros_like(st["ctx"]), width=width)
        else:
            Hq, words = case["Hq"], _pages(max(new), 32)
            depth, sees = _trees(random.Random(seed), new)
            bits = np.array([[(a >> 32 * w) & 0xffffffff for w in range(words)] for a in sees], np.uint32)
            st.update(offsets=i32(np.cumsum([0] + new).tolist()), mask=torch.from_numpy(bits.view(np.int32)).cuda(), words=words,
                      positions=i32((np.array(ctx)[seq] + np.array(depth)).tolist()), q=rows(tokens, Hq * D), tokens=tokens, most_new=max(new),
                      longest=max(after), o=torch.zeros(tokens, Hq, D, device="cuda", dtype=dt), lse=torch.zeros(tokens, Hq, device="cuda"))
    if own:
        fa = framework()
        st["batch"] = fa.PagedBatch(S, page, pool, most, page_tables=st["table"], page_counts=st["held"], context_lens=st["ctx"],
                                    free_pages=st["free"], free_count=st["free_count"])
        if op == "tree":
            dtype = fa.BF16 if case["dtype"] == "bf16" else fa.F32
            st["out"] = context().create_decode_output_buffer(dtype, tokens, case["Hq"], case["D"])
            st["o"], st["lse"] = context().split_decode_output(st["out"], dtype, tokens, case["Hq"], case["D"])
            st["cfg"] = fa.config(True)
    return st


# ---- one pass ------------------------------------------------------------------------------------

def run(st):
    if own:
        return _run_own(st)
    return {"reserve": _reserve, "release": _release, "write": _write, "accept": _accept, "tree": _tree}[st["op"]](st)


def _run_own(st):
    ctx, c, batch = context(), st["case"], st["batch"]
    if st["op"] == "reserve":
        ctx.paged_batch_reserve(batch, st["new"], st["tokens"], st["offsets"], st["slots"], st["positions"],
                                page_counts_out=st["held_out"], free_count_out=st["free_count_out"])
        return dict(table=st["table"], held=st["held_out"], free_count=st["free_count_out"], offsets=st["offsets"], slots=st["slots"],
                    positions=st["positions"])
    if st["op"] == "release":
        ctx.paged_batch_release(batch, st["new"], page_counts_out=st["held_out"], free_count_out=st["free_count_out"])
        return dict(free=st["free"], held=st["held_out"], free_count=st["free_count_out"])
    if st["op"] == "write":
        ctx.paged_kv_write(c["Hkv"], c["D"], st["slots"], st["positions"], THETA, st["k_new"], st["v_new"], st["k"], st["v"])
        return dict(k=st["k"], v=st["v"])
    if st["op"] == "accept":
        ctx.paged_kv_accept(batch, c["Hkv"], c["D"], st["path"], st["takes"], st["ctx_out"], st["k"], st["v"])
        return dict(k=st["k"], v=st["v"], ctx=st["ctx_out"])
    ctx.decode_paged_tree(batch, c["Hq"], c["Hkv"], c["D"], st["most_new"], st["longest"], st["offsets"], st["positions"], st["mask"],
                          st["cfg"], THETA, st["q"], st["k"], st["v"], st["out"])
    return dict(o=st["o"], lse=st["lse"])


def _reserve(st):
    page = st["case"]["page"]
    L, N, H, table, free = st["ctx"].long(), st["new"].long(), st["held"].long(), st["table"], st["free"].long()
    f, S = st["free_count"].long(), st["case"]["S"]
    need = ((L + N + page - 1) // page - H).clamp(min=0)
    upto = need.cumsum(0)
    given = torch.where((need == 0) | (upto <= f), need, torch.zeros_like(need))
    ok = (need == 0) | (upto <= f)
    col = torch.arange(st["most"], device=L.device)[None, :]
    fresh = (col >= H[:, None]) & (col < (H + given)[:, None])
    where = f - 1 - ((upto - need)[:, None] + col - H[:, None])
    table = torch.where(fresh, free[where.clamp(0, st["pool"] - 1)].int(), table)
    offsets = torch.cat([N.new_zeros(1), N.cumsum(0)])
    seq = torch.repeat_interleave(torch.arange(S, device=L.device), N, output_size=st["tokens"])
    at = L[seq] + torch.arange(st["tokens"], device=L.device) - offsets[seq]
    slots = torch.where(ok[seq], table[seq, at // page].long() * page + at % page, torch.full_like(at, -1))
    return dict(table=table, held=(H + given).int(), free_count=(f - given.sum()).int(), offsets=offsets.int(), slots=slots.int(),
                positions=torch.where(ok[seq], at, torch.zeros_like(at)).int())


def _release(st):
    page = st["case"]["page"]
    keep, H, table, f = st["new"].long(), st["held"].long(), st["table"], st["free_count"].long()
    left = torch.minimum(H, (keep.clamp(min=0) + page - 1) // page)
    gone = H - left
    upto = gone.cumsum(0)
    col = torch.arange(st["most"], device=H.device)[None, :]
    goes = (col >= left[:, None]) & (col < H[:, None])
    to = f + (upto - gone)[:, None] + (H[:, None] - 1 - col)
    free = st["free"].clone()
    free[to[goes]] = table[goes]
    return dict(free=free, held=left.int(), free_count=(f + gone.sum()).int())


def _rotated(x, positions, D):
    """Neighbouring pairs of each head's slice turned by position * theta^(-2 j / D); angles in 64 bits, the rest in 32."""
    freq = THETA ** (-2.0 * torch.arange(D // 2, device=x.device, dtype=torch.float64) / D)
    angle = positions.double()[:, None] * freq
    c, s = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    x = x.float().view(x.shape[0], -1, D // 2, 2)
    a, b = x[..., 0], x[..., 1]
    return torch.stack([a * c - b * s, a * s + b * c], -1).view(x.shape[0], -1, D)


def _write(st):
    k, v, D, slots = st["k"], st["v"], st["case"]["D"], st["slots"].long()
    k[slots] = _rotated(st["k_new"], st["positions"], D).view(len(slots), -1).to(k.dtype)
    v[slots] = st["v_new"]
    return dict(k=k, v=v)


def _accept(st):
    c, L, path, takes = st["case"], st["ctx"].long(), st["path"].long(), st["takes"].long()
    j = torch.arange(st["width"], device=L.device)[None, :]
    on = j < takes[:, None]
    rows = lambda at: (st["table"].gather(1, (at // c["page"]).clamp(0, st["most"] - 1)).long() * c["page"] + at % c["page"])[on]  # noqa: E731
    src, dst = rows(L[:, None] + path.clamp(min=0)), rows(L[:, None] + j)
    st["k"][dst] = st["k"][src]
    st["v"][dst] = st["v"][src]
    return dict(k=st["k"], v=st["v"], ctx=(L + takes).int())


def _tree(st):
    c = st["case"]
    S, Hq, Hkv, D, page, n, most = c["S"], c["Hq"], c["Hkv"], c["D"], c["page"], st["most_new"], st["longest"]
    G, dev = Hq // Hkv, st["q"].device
    L, off = st["ctx"].long(), st["offsets"].long()
    N = off[1:] - off[:-1]
    q = _rotated(st["q"], st["positions"], D) / math.sqrt(D)
    i = torch.arange(n, device=dev)[None, :]
    on = i < N[:, None]
    row = (off[:-1, None] + i).clamp(max=st["tokens"] - 1)
    q = (q[row] * on[:, :, None, None]).view(S, n, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, n * G, D)
    t = torch.arange(most, device=dev)[None, :].expand(S, most)
    live = t < (L + N)[:, None]
    at = st["table"].long().gather(1, torch.where(live, t // page, torch.zeros_like(t))).clamp(min=0) * page + t % page
    rows = lambda x: (x[at].float() * live[:, :, None]).view(S, most, Hkv, D).permute(0, 2, 1, 3)  # noqa: E731
    node = (t - L[:, None]).clamp(0, 32 * st["words"] - 1)
    word = st["mask"][row].gather(2, (node // 32)[:, None, :].expand(S, n, most))
    sees = ((word >> (node % 32)[:, None, :].int()) & 1).bool() | (t < L[:, None])[:, None, :]
    sees = (sees & live[:, None, :])[:, None, :, None, :]
    x = (q @ rows(st["k"]).transpose(2, 3)).view(S, Hkv, n, G, most).masked_fill(~sees, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    o = (x.view(S, Hkv, n * G, most) @ rows(st["v"])).view(S, Hkv, n, G, D) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + total.log())[..., 0]
    o, lse = o.permute(0, 2, 1, 3, 4).reshape(S, n, Hq, D)[on], lse.permute(0, 2, 1, 3).reshape(S, n, Hq)[on]
    return dict(o=o.to(st["q"].dtype), lse=lse)


# ---- floors and the definition in 64 bits --------------------------------------------------------

def work(case):
    ctx, new = _lengths(case)
    page, S = case["page"], case["S"]
    if case["op"] == "reserve":
        took = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(ctx, new))
        return dict(bytes=16 * S + 8 * sum(new) + 8 * took, flops=0)
    if case["op"] == "release":
        gone = sum(_pages(a, page) - min(_pages(a, page), _pages(b, page)) for a, b in zip(ctx, new))
        return dict(bytes=12 * S + 8 * gone, flops=0)
    size = 2 if case["dtype"] == "bf16" else 4
    line = 2 * case["Hkv"] * case["D"] * size
    if case["op"] == "write":
        return dict(bytes=sum(new) * (2 * line + 8), flops=3 * sum(new) * case["Hkv"] * case["D"])
    if case["op"] == "accept":
        # a third of a path or so stays where it is; which nodes move is in the inputs, so all count
        return dict(bytes=sum(_takes(case, new)) * (2 * line + 4) + 12 * S, flops=0)
    Hq, D = case["Hq"], case["D"]
    return dict(bytes=sum(a + b for a, b in zip(ctx, new)) * line + sum(new) * Hq * (2 * D * size + 4) + sum(new) * 8,
                flops=4 * D * Hq * sum(b * (a + 1) for a, b in zip(ctx, new)))


def exact(case, seed):
    kept, st = own, None
    globals()["own"] = False
    try:
        st = prepare(case, seed)
    finally:
        globals()["own"] = kept
    ctx, new = _lengths(case)
    page, op = case["page"], case["op"]
    table = st["table"].cpu().numpy()
    if op == "reserve":
        f, free, held = int(st["free_count"]), st["free"].cpu().numpy(), st["held"].cpu().numpy().copy()
        slots, positions = [], []
        for s in range(case["S"]):
            want = _pages(ctx[s] + new[s], page)
            while held[s] < want:  # the pool of a case has the pages
                f -= 1
                table[s, held[s]] = free[f]
                held[s] += 1
            at = np.arange(ctx[s], ctx[s] + new[s])
            slots.append(table[s, at // page] * page + at % page)
            positions.append(at)
        return dict(table=table, held=held, free_count=np.array([f], np.int32), offsets=np.cumsum([0] + new).astype(np.int32),
                    slots=np.concatenate(slots).astype(np.int32), positions=np.concatenate(positions).astype(np.int32))
    if op == "release":
        f, free, held = int(st["free_count"]), st["free"].cpu().numpy(), st["held"].cpu().numpy().copy()
        for s in range(case["S"]):
            while held[s] > _pages(new[s], page):
                held[s] -= 1
                free[f] = table[s, held[s]]
                f += 1
        return dict(free=free, held=held, free_count=np.array([f], np.int32))
    k, v, D = st["k"].double(), st["v"].double(), case["D"]
    freq = torch.tensor([THETA ** (-2.0 * j / D) for j in range(D // 2)], dtype=torch.float64, device="cuda")

    def turned(x, positions):
        z = torch.view_as_complex(x.double().reshape(x.shape[0], -1, D // 2, 2).contiguous())
        by = positions.double()[:, None] * freq
        return torch.view_as_real(z * torch.polar(torch.ones_like(by), by)[:, None, :]).reshape(x.shape[0], -1, D)

    if op == "write":
        at = st["slots"].long()
        k.index_copy_(0, at, turned(st["k_new"], st["positions"]).reshape(len(at), -1))
        v.index_copy_(0, at, st["v_new"].double())
        return dict(k=k, v=v)
    line = lambda s, t: int(table[s, t // page]) * page + t % page  # noqa: E731
    if op == "accept":
        path, takes = st["path"].cpu().numpy(), st["takes"].tolist()
        src = [line(s, ctx[s] + int(path[s, j])) for s in range(case["S"]) for j in range(takes[s])]
        dst = [line(s, ctx[s] + j) for s in range(case["S"]) for j in range(takes[s])]
        if src:  # no row of a path is both a source and another one's destination
            k[dst], v[dst] = k[src], v[src]
        return dict(k=k, v=v, ctx=np.array([a + b for a, b in zip(ctx, takes)], np.int32))
    Hq, Hkv = case["Hq"], case["Hkv"]
    q, words = turned(st["q"], st["positions"]), st["mask"].cpu().numpy().view(np.uint32)
    o, lse, first = [], [], 0
    for a, n, pages in zip(ctx, new, table):
        at = np.arange(a + n)
        at = torch.from_numpy(pages[at // page].astype(np.int64) * page + at % page).cuda()
        bits = np.unpackbits(words[first:first + n].view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
        seen = torch.from_numpy(np.concatenate([np.ones((n, a), bool), bits], 1)).cuda()
        kk = k[at].view(a + n, Hkv, D).repeat_interleave(Hq // Hkv, 1)
        vv = v[at].view(a + n, Hkv, D).repeat_interleave(Hq // Hkv, 1)
        x = torch.einsum("nhd,thd->hnt", q[first:first + n], kk) / math.sqrt(D)
        x = x.masked_fill(~seen, -math.inf)
        lse.append(torch.logsumexp(x, -1).T)
        o.append(torch.einsum("hnt,thd->nhd", torch.softmax(x, -1), vv))
        first += n
    return dict(o=torch.cat(o), lse=torch.cat(lse))
