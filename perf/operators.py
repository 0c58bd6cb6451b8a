"""What the speculative-decoding operators are measured on.

Attention for trees of drafted tokens over the paged cache, verification of
the drafts against the target's probabilities, and the cache's page moves
(keeping an accepted path, copying pages).  Every case has its plain form in
elementary torch operations (``own`` false) and the framework's calls
(``own`` true) on the same inputs.

Trees: the rows of sequence s are ``q_start[s] .. q_start[s] + q_len[s] - 1``;
row i of them is node i, node 0 the root (the last accepted token), and
``parents`` holds each node's parent inside its sequence (-1 for the root).
Node i's keys and values lie at position ``ctx_len - q_len + i``.
"""
from __future__ import annotations

import random

import numpy as np
import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------- cases


def listed():
    return [
        # a lone chat request on the smallest model, a short chain of drafts: latency only
        dict(name="attn_one_short", op="attn", n=1, hq=14, hkv=2, hd=64, bs=16, nodes=5, branch=1,
             ctx_lo=200, ctx_hi=300),
        # a batch of chat requests, a chain of drafts each: the cache's bytes
        dict(name="attn_batch_chain", op="attn", n=32, hq=40, hkv=8, hd=128, bs=16, nodes=6,
             branch=1, ctx_lo=500, ctx_hi=4000),
        # some requests with a tree of drafts each, ragged contexts
        dict(name="attn_batch_tree", op="attn", n=16, hq=40, hkv=8, hd=128, bs=16, nodes=25,
             branch=4, ctx_lo=300, ctx_hi=6000),
        # few long documents on the widest heads, the largest trees: many rows for each key read
        dict(name="attn_long_wide_tree", op="attn", n=4, hq=64, hkv=8, hd=128, bs=32, nodes=64,
             branch=4, ctx_lo=12000, ctx_hi=20000),
        # one request, greedy sampling: latency only
        dict(name="greedy_one", op="greedy", n=1, nodes=16, branch=3, depth=6, vocab=151936),
        # a serving batch, greedy sampling
        dict(name="greedy_batch", op="greedy", n=128, nodes=48, branch=4, depth=8, vocab=152064),
        # one request, a tree of drafts picked outright (no draft distribution)
        dict(name="verify_one_picked", op="verify", n=1, nodes=26, branch=4, depth=6,
             vocab=151936, dist=False),
        # a serving batch, chains sampled from a draft model
        dict(name="verify_batch_chain", op="verify", n=64, nodes=6, branch=1, depth=6,
             vocab=152064, dist=True),
        # some requests, trees sampled from a draft model without replacement
        dict(name="verify_batch_tree", op="verify", n=8, nodes=40, branch=4, depth=6,
             vocab=152064, dist=True),
        # the accepted paths of a batch, all layers
        dict(name="keep_batch", op="keep", n=64, layers=48, hkv=8, hd=128, bs=16, nodes=25,
             accepted=5, blocks=4),
        # one fork: its half-filled last page, all layers of the smallest model
        dict(name="copy_one_fork", op="copy", n=1, layers=24, hkv=2, hd=64, bs=16),
        # forks and moves of many pages, all layers
        dict(name="copy_many", op="copy", n=200, layers=48, hkv=8, hd=128, bs=16),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "greedy", "verify", "verify", "keep", "copy"])
    if op == "attn":
        hq, hkv, hd = rng.choice([(14, 2, 64), (40, 8, 128), (64, 8, 128), (20, 4, 128), (7, 1, 64)])
        nodes = _log(rng, 1, 64)
        n = _log(rng, 1, 64)
        # the largest listed case holds 80000 cached tokens of 512 rows a kv head
        hi = _log(rng, 20, max(21, min(20000, 80000 // n)))
        return dict(op=op, n=n, hq=hq, hkv=hkv, hd=hd, bs=rng.choice([16, 32]), nodes=nodes,
                    branch=rng.choice([1, 2, 4, 8]), ctx_lo=max(1, hi // rng.choice([1, 2, 10])),
                    ctx_hi=hi)
    vocab = rng.choice([151936, 152064, _log(rng, 100, 152064)])
    if op == "greedy":
        return dict(op=op, n=_log(rng, 1, 128), nodes=_log(rng, 1, 64),
                    branch=rng.choice([1, 2, 4]), depth=rng.randint(2, 8), vocab=vocab)
    if op == "verify":
        nodes = _log(rng, 1, 64)
        return dict(op=op, n=_log(rng, 1, max(2, 384 // nodes)), nodes=nodes,
                    branch=rng.choice([1, 2, 4]), depth=rng.randint(2, 8), vocab=vocab,
                    dist=rng.random() < 0.6)
    layers, hkv, hd = rng.choice([(24, 2, 64), (48, 8, 128), (48, 4, 128), (80, 8, 128)])
    cap = max(1, 9600 * 1024 // (layers * hkv * hd))
    if op == "keep":
        return dict(op=op, n=_log(rng, 1, min(64, max(2, cap // 4))), layers=layers, hkv=hkv, hd=hd,
                    bs=rng.choice([16, 32]), nodes=_log(rng, 2, 60), accepted=rng.randint(1, 8),
                    blocks=4)
    return dict(op=op, n=_log(rng, 1, min(200, cap)), layers=layers, hkv=hkv, hd=hd, bs=16)


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """Node counts and context lengths of a case's sequences (the same for every seed)."""
    r = random.Random("lengths %d %d" % (case["n"], case["nodes"]))
    n, q = case["n"], case["nodes"]
    q_len = [q if i == 0 else r.randint(max(1, q - q // 4), q) for i in range(n)]
    if "ctx_hi" not in case:
        return q_len, None
    lo, hi = case["ctx_lo"], case["ctx_hi"]
    return q_len, [(hi if i == 0 else r.randint(lo, hi)) + q_len[i] for i in range(n)]


def _tree(r, nodes, branch, depth):
    """Parents of a random tree in node order: every node has at most ``branch`` children and
    lies at most ``depth`` levels below the root."""
    parent, level, kids = [-1], [0], [0]
    open_ = [0]
    for i in range(1, nodes):
        p = i - 1 if branch == 1 else r.choice(open_)
        if branch == 1 and level[p] >= depth:
            p = r.choice(open_)
        parent.append(p)
        level.append(level[p] + 1)
        kids.append(0)
        kids[p] += 1
        if kids[p] >= branch and len(open_) > 1 and p in open_:
            open_.remove(p)
        if level[i] < depth:
            open_.append(i)
    return parent, level


def _masks(parent):
    """Ancestor bits of every node, itself included (at most 64 nodes)."""
    m = [0] * len(parent)
    for i, p in enumerate(parent):
        m[i] = (m[p] if p >= 0 else 0) | (1 << i)
    return m


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(lengths):
    return [0] + np.cumsum(lengths).tolist()[:-1]


def _blocks(r, need, extra):
    """Disjoint random block lists of the given lengths, padded to a table with -1."""
    ids = list(range(sum(need) + extra))
    r.shuffle(ids)
    width, at, table = max(need), 0, []
    for k in need:
        table.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    return table, len(ids)


def prepare(case, seed):
    r = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"attn": _prepare_attn, "greedy": _prepare_drafts, "verify": _prepare_drafts,
            "keep": _prepare_keep, "copy": _prepare_copy}[case["op"]](case, r, g)


def _prepare_attn(case, r, g):
    q_len, ctx = _lengths(case)
    hq, hkv, hd, bs = case["hq"], case["hkv"], case["hd"], case["bs"]
    table, n_blocks = _blocks(r, [-(-c // bs) for c in ctx], 3)
    masks = []
    for k in q_len:
        masks += _masks(_tree(r, k, case["branch"], 64)[0])
    rows = sum(q_len)
    return dict(
        op="attn", hq=hq, hkv=hkv, hd=hd, bs=bs, max_q=max(q_len), max_ctx=max(ctx),
        ctx_total=sum(ctx),
        # a query's scores spread over a few units, as trained heads' do
        q=(torch.randn(rows, hq * hd, generator=g, device=DEV) * 1.5).bfloat16(),
        out=torch.zeros(rows, hq * hd, dtype=torch.bfloat16, device=DEV),
        pool=torch.randn(n_blocks, 2, hkv, bs, hd, generator=g, device=DEV, dtype=torch.bfloat16),
        bt=_ints(table), q_start=_ints(_starts(q_len)), q_len=_ints(q_len), ctx=_ints(ctx),
        # bit 63 of the 64-bit words is their sign
        mask=torch.from_numpy(np.array(masks, dtype=np.uint64).view(np.int64)).to(DEV)[:, None])


def _prepare_drafts(case, r, g):
    q_len, _ = _lengths(case)
    q_start = _starts(q_len)
    n, V, rows = case["n"], case["vocab"], sum(q_len)
    parents, rank, row_of_parent = [], [], []
    inner = {}                      # rows with children -> row of their draft distribution
    for s, k in enumerate(q_len):
        par, _ = _tree(r, k, case["branch"], case["depth"])
        kids = [0] * k
        for p in par:
            row_of_parent.append(q_start[s] + max(p, 0))
            rank.append(kids[p] if p >= 0 else 0)
            if p >= 0:
                kids[p] += 1
                inner.setdefault(q_start[s] + p, len(inner))
        parents += par
    st = dict(op=case["op"], max_q=max(q_len), branch=max(rank) + 1, parents=_ints(parents),
              q_start=_ints(q_start), q_len=_ints(q_len),
              n_accepted=torch.zeros(n, dtype=torch.int32, device=DEV),
              path=torch.zeros(n, min(case["depth"], max(q_len) - 1) + 1, dtype=torch.int32,
                               device=DEV),
              next_ids=torch.zeros(n, dtype=torch.int32, device=DEV))
    if case["op"] == "greedy":
        target = [r.randrange(V) for _ in range(rows)]
        # most first children are what the target chose, some second ones too
        st["ids"] = _ints([target[p] if r.random() < (0.75, 0.4, 0.1, 0.1)[min(k, 3)] else r.randrange(V)
                           for p, k in zip(row_of_parent, rank)])
        st["target_ids"] = _ints(target)
        return st
    # peaked distributions, as language models' are; the draft's logits are the target's, disturbed
    logits = torch.randn(rows, V, generator=g, device=DEV) * 2.5
    st["probs"] = torch.softmax(logits, -1)
    keys = list(inner) or [0]
    d = logits[torch.tensor(keys, device=DEV)]
    del logits
    d += torch.randn(d.shape, generator=g, device=DEV) * 0.7
    d = torch.softmax(d, -1)
    # the tokens of a node's children: drawn without replacement, or the most probable ones
    score = d.log()
    if case["dist"]:
        score -= torch.empty_like(d).exponential_(generator=g).log_()
    top = score.topk(min(max(rank) + 1, V), -1).indices
    del score
    at = torch.tensor([inner.get(p, 0) for p in row_of_parent], device=DEV)
    st["ids"] = top[at, torch.tensor(rank, device=DEV).clamp_(max=top.shape[1] - 1)].int()
    st["uniforms"] = torch.rand(rows, generator=g, device=DEV)
    st["draft_probs"] = d if case["dist"] else None
    st["draft_rows"] = _ints([inner.get(i, -1) for i in range(rows)]) if case["dist"] else None
    return st


def _prepare_keep(case, r, g):
    q_len, _ = _lengths(case)
    n, bs = case["n"], case["bs"]
    need = [case["blocks"] + -(-k // bs) for k in q_len]
    table, n_blocks = _blocks(r, need, 2)
    ctx = [r.randint(k, b * bs) for k, b in zip(q_len, need)]
    width = min(case["accepted"], case["nodes"] - 1) + 1
    accepted = [min(width - 1, k - 1) if i == 0 else r.randint(0, min(width, k) - 1)
                for i, k in enumerate(q_len)]
    path = [[0] + sorted(r.sample(range(1, k), a)) + [-1] * (width - 1 - a)
            for k, a in zip(q_len, accepted)]
    return dict(op="keep", bs=bs, bt=_ints(table), q_len=_ints(q_len), ctx=_ints(ctx),
                path=_ints(path), n_accepted=_ints(accepted),
                pools=torch.randn(case["layers"], n_blocks, 2, case["hkv"], bs, case["hd"],
                                  generator=g, device=DEV, dtype=torch.bfloat16))


def _prepare_copy(case, r, g):
    n = case["n"]
    ids = list(range(2 * n + 3))
    r.shuffle(ids)
    # a page may be copied several times; every destination is a page of its own
    pairs = [[ids[r.randrange(max(1, n // 2), n + 1) - 1], ids[n + i]] for i in range(n)]
    return dict(op="copy", pairs=_ints(pairs),
                pools=torch.randn(case["layers"], len(ids), 2, case["hkv"], case["bs"], case["hd"],
                                  generator=g, device=DEV, dtype=torch.bfloat16))


# ------------------------------------------------------------------ passes


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "greedy": _plain_greedy, "verify": _plain_verify,
            "keep": _plain_keep, "copy": _plain_copy}[state["op"]](state)


def _run_own(st):
    from tinybatch_b200 import ops
    op = st["op"]
    if op == "attn":
        ops.paged_attention_tree(
            st["q"], st["out"], st["pool"], n_q_heads=st["hq"], n_kv_heads=st["hkv"],
            head_dim=st["hd"], block_size=st["bs"], block_tables=st["bt"], q_start=st["q_start"],
            q_len=st["q_len"], ctx_len=st["ctx"], tree_mask=st["mask"], max_q=st["max_q"],
            max_ctx=st["max_ctx"], ctx_total=st["ctx_total"])
        return st["out"]
    if op == "keep":
        ops.keep_kv_path(st["pools"], block_tables=st["bt"], q_len=st["q_len"], ctx_len=st["ctx"],
                         path=st["path"], n_accepted=st["n_accepted"])
        return st["pools"]
    if op == "copy":
        ops.copy_kv_blocks(st["pools"], st["pairs"])
        return st["pools"]
    if op == "greedy":
        ops.verify_drafts_greedy(st["ids"], st["parents"], st["q_start"], st["q_len"],
                                 st["target_ids"], st["n_accepted"], st["path"], st["next_ids"],
                                 max_q=st["max_q"])
    else:
        ops.verify_drafts(st["ids"], st["parents"], st["q_start"], st["q_len"], st["probs"],
                          st["uniforms"], st["n_accepted"], st["path"], st["next_ids"],
                          draft_probs=st["draft_probs"], draft_rows=st["draft_rows"],
                          max_q=st["max_q"])
    return st["n_accepted"], st["path"], st["next_ids"]


def _plain_attn(st):
    """Whole contexts gathered from the pages, scores of every (node, key), softmax in 32 bits."""
    hq, hkv, hd, Q = st["hq"], st["hkv"], st["hd"], st["max_q"]
    n, G = st["q_len"].shape[0], hq // hkv
    kv = st["pool"][st["bt"].clamp(min=0).long()]             # [n, pages, 2, hkv, bs, hd]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, n, hkv, 1, -1, hd).float()
    node = torch.arange(Q, device=DEV)
    real = node < st["q_len"][:, None]                        # [n, Q]
    row = torch.where(real, st["q_start"][:, None] + node, 0).long()
    q = st["q"][row].view(n, Q, hkv, G, hd).permute(0, 2, 3, 1, 4).float()
    s = torch.matmul(q * hd ** -0.5, kv[0].transpose(-1, -2))  # [n, hkv, G, Q, keys]
    pos = torch.arange(kv.shape[4], device=DEV)
    j = pos - (st["ctx"] - st["q_len"])[:, None]              # draft index of a key, < 0 in the prefix
    bits = st["mask"][row, 0]
    seen = (j[:, None] < 0) | ((bits[:, :, None] >> j.clamp(0, 63)[:, None]) & 1).bool()
    seen &= (j < st["q_len"][:, None])[:, None]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, kv[1]) / torch.where(total > 0, total, 1)
    o = o.permute(0, 3, 1, 2, 4).reshape(n * Q, hq * hd)
    # rows of short sequences repeat row 0's place: give every row its own source instead
    seq = torch.searchsorted(st["q_start"], torch.arange(st["q"].shape[0], device=DEV,
                                                         dtype=torch.int32), right=True) - 1
    src = seq * Q + torch.arange(st["q"].shape[0], device=DEV) - st["q_start"][seq]
    return o[src].bfloat16()


def _grid(st):
    """Row of node j of sequence s, which of them are real, and each node's children in node
    order (the sequence's node count where there is none)."""
    Q, m = st["max_q"], st["branch"]
    node = torch.arange(Q, device=DEV)
    real = node < st["q_len"][:, None]
    row = torch.where(real, st["q_start"][:, None] + node, 0).long()
    par = torch.where(real, st["parents"][row], -2)
    kids = torch.where(par[:, None, :] == node[:, None], node, Q).sort(-1).values[..., :m]
    return row, kids


def _plain_greedy(st):
    row, kids = _grid(st)
    n, Q = row.shape
    P = st["path"].shape[1]
    kid_row = torch.gather(row, 1, kids.clamp(max=Q - 1).view(n, -1)).view(kids.shape)
    hit = (kids < Q) & (st["ids"][kid_row] == st["target_ids"][row][..., None])
    nxt = torch.where(hit, kids, Q).amin(-1)                  # [n, Q]: node after each node
    nxt = torch.cat([nxt, torch.full_like(nxt[:, :1], Q)], 1)
    cur, path = torch.zeros(n, dtype=torch.long, device=DEV), []
    path.append(cur)
    for _ in range(P - 1):
        cur = torch.gather(nxt, 1, cur[:, None])[:, 0]
        path.append(cur)
    path = torch.stack(path, 1)
    took = (path < Q).sum(1) - 1
    last = torch.gather(path, 1, took[:, None])
    next_ids = st["target_ids"][torch.gather(row, 1, last)[:, 0]]
    return took.int(), torch.where(path < Q, path, -1).int(), next_ids


def _plain_verify(st):
    row, kids = _grid(st)
    n, Q = row.shape
    P, V = st["path"].shape[1], st["probs"].shape[1]
    u = st["uniforms"].double()
    cur = torch.zeros(n, dtype=torch.long, device=DEV)
    walking = torch.ones(n, dtype=torch.bool, device=DEV)
    final = torch.zeros(n, V, dtype=torch.float64, device=DEV)
    path = [cur]
    for level in range(P):
        at = torch.gather(row, 1, cur[:, None])[:, 0]
        r = st["probs"][at].double()
        found = torch.full_like(cur, -1)
        if st["draft_rows"] is not None:
            d_row = st["draft_rows"][at].long()
            has = d_row >= 0
            d = st["draft_probs"][d_row.clamp(min=0)].double()
        gone = torch.zeros(n, dtype=torch.float64, device=DEV)
        for k in range(st["branch"] if level < P - 1 else 0):
            kid = kids[torch.arange(n, device=DEV), cur, k]
            kid_row = torch.gather(row, 1, kid.clamp(max=Q - 1)[:, None])[:, 0]
            x = st["ids"][kid_row].long()[:, None]
            testing = walking & (kid < Q) & (found < 0)
            rx = torch.gather(r, 1, x)[:, 0]
            picked = (rx > 0) & (u[kid_row] * (1 - gone) < rx)
            if st["draft_rows"] is None:
                ok = picked
                off = testing & ~ok
                gone = torch.where(off, gone + rx, gone)
                r = torch.where(off[:, None], r.scatter(1, x, 0.0), r)
            else:
                dx0 = torch.gather(d, 1, x)[:, 0]
                left = 1 - gone
                scale = torch.where(left > 0, 1 / left, 0)
                ok = torch.where(has, (dx0 * scale > 0) & (u[kid_row] * (dx0 * scale) < rx), picked)
                off = testing & ~ok & has & (dx0 * scale > 0)
                rest = (r - d * scale[:, None]).clamp(min=0)
                z = rest.sum(1)
                r = torch.where((off & (z > 0))[:, None], rest / z[:, None], r)
                lone = testing & ~ok & ~has
                gone = torch.where(off, gone + dx0, torch.where(lone, gone + rx, gone))
                d = torch.where(off[:, None], d.scatter(1, x, 0.0), d)
                r = torch.where(lone[:, None], r.scatter(1, x, 0.0), r)
            found = torch.where(testing & ok, kid, found)
        stop = walking & (found < 0)
        final = torch.where(stop[:, None], r, final)
        walking &= found >= 0
        cur = torch.where(walking, found, cur)
        if level < P - 1:
            path.append(torch.where(walking, found, -1))
    path = torch.stack(path, 1)
    cdf = final.cumsum(1)
    t = u[st["q_start"].long()] * cdf[:, -1]
    pick = torch.searchsorted(cdf, t[:, None], right=True)[:, 0].clamp(max=V - 1)
    next_ids = torch.where(cdf[:, -1] > 0, pick, -1)
    return ((path >= 0).sum(1) - 1).int(), path.int(), next_ids.int()


def _plain_keep(st):
    bs, path = st["bs"], st["path"]
    j = torch.arange(path.shape[1], device=DEV)
    base = (st["ctx"] - st["q_len"])[:, None].long()
    moved = j <= st["n_accepted"][:, None]
    src = base + torch.where(moved, path, 0)                  # the others: the root onto itself
    dst = base + torch.where(moved, j, 0)
    bt = st["bt"].long()
    sb, ss = torch.gather(bt, 1, src // bs).view(-1), (src % bs).view(-1)
    db, ds = torch.gather(bt, 1, dst // bs).view(-1), (dst % bs).view(-1)
    st["pools"][:, db, :, :, ds] = st["pools"][:, sb, :, :, ss]
    return st["pools"]


def _plain_copy(st):
    src, dst = st["pairs"].long().unbind(1)
    st["pools"][:, dst] = st["pools"][:, src]
    return st["pools"]


# -------------------------------------------------------------------- work


def work(case):
    op, n = case["op"], case["n"]
    if op == "attn":
        q_len, ctx = _lengths(case)
        rows = sum(q_len)
        r = random.Random("work")
        pairs = 0
        for k, c in zip(q_len, ctx):
            seen = sum(bin(m).count("1") for m in _masks(_tree(r, k, case["branch"], 64)[0]))
            pairs += k * (c - k) + seen
        kv = sum(ctx) * case["hkv"] * case["hd"] * 4
        return dict(bytes=kv + rows * (4 * case["hq"] * case["hd"] + 8),
                    flops=4 * case["hd"] * case["hq"] * pairs)
    if op == "greedy":
        return dict(bytes=sum(_lengths(case)[0]) * 12 + n * (12 + 4 * (case["depth"] + 1)),
                    flops=0)
    if op == "verify":
        # one target row a sequence and, with draft distributions, the draft row it is lessened by
        rows = (2 if case["dist"] and case["nodes"] > 1 else 1) * n
        return dict(bytes=rows * case["vocab"] * 4 + sum(_lengths(case)[0]) * 24, flops=3 * rows * case["vocab"])
    page = case["layers"] * 2 * case["hkv"] * case["hd"] * 2
    if op == "keep":
        a = min(case["accepted"], case["nodes"] - 1)
        # all of the first sequence's path, half of it on average in the others
        return dict(bytes=2 * page * max(1, int(a + (n - 1) * a / 2)), flops=0)
    return dict(bytes=2 * page * case["bs"] * n, flops=0)


# ------------------------------------------------------------------- exact


def exact(case, seed):
    st = prepare(case, seed)
    return {"attn": _exact_attn, "greedy": _exact_drafts, "verify": _exact_drafts,
            "keep": _exact_keep, "copy": _exact_copy}[case["op"]](st)


def _exact_attn(st):
    """Sequence by sequence and kv head by kv head, from the definition, in 64 bits."""
    hd, bs = st["hd"], st["bs"]
    G = st["hq"] // st["hkv"]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device=DEV)
    words = st["mask"][:, 0].tolist()
    for s, (a, k, c) in enumerate(zip(st["q_start"].tolist(), st["q_len"].tolist(),
                                      st["ctx"].tolist())):
        pages = st["bt"][s, :-(-c // bs)].tolist()
        hidden = torch.tensor([[not (words[a + i] >> j) & 1 for j in range(k)] for i in range(k)],
                              device=DEV)
        for h in range(st["hkv"]):
            k_, v_ = (torch.cat([st["pool"][b, w, h] for b in pages])[:c].double() for w in (0, 1))
            for g in range(h * G, h * G + G):
                x = st["q"][a:a + k, g * hd:(g + 1) * hd].double() @ k_.T / hd ** 0.5
                x[:, c - k:][hidden] = -torch.inf
                out[a:a + k, g * hd:(g + 1) * hd] = torch.softmax(x, -1) @ v_
    return out


def _exact_drafts(st):
    """One sequence after another, one node after another."""
    ids, parents = st["ids"].tolist(), st["parents"].tolist()
    greedy = st["op"] == "greedy"
    if greedy:
        target = st["target_ids"].tolist()
    else:
        u = st["uniforms"].double().tolist()
        d_rows = st["draft_rows"].tolist() if st["draft_rows"] is not None else [-1] * len(ids)
    width = st["path"].shape[1]
    took, paths, nexts = [], [], []
    for a, k in zip(st["q_start"].tolist(), st["q_len"].tolist()):
        path, moved = [0], True
        while moved:
            moved, c = False, path[-1]
            kids = [i for i in range(c + 1, k) if parents[a + i] == c] if len(path) < width else []
            if greedy:
                good = [i for i in kids if ids[a + i] == target[a + c]]
                if good:
                    path.append(good[0])
                    moved = True
                continue
            r = st["probs"][a + c].double()
            d = st["draft_probs"][d_rows[a + c]].double() if d_rows[a + c] >= 0 else None
            left = 1.0
            for i in kids:
                x = ids[a + i]
                if d is None:
                    if 0 < float(r[x]) > u[a + i] * left:
                        path.append(i)
                        moved = True
                        break
                    left -= float(r[x])
                    r = r.clone()
                    r[x] = 0
                    continue
                share = float(d[x]) / left if left > 0 else 0.0
                if share <= 0:
                    continue
                if u[a + i] * share < float(r[x]):
                    path.append(i)
                    moved = True
                    break
                rest = torch.relu(r - d / left)
                if float(rest.sum()) > 0:
                    r = rest / rest.sum()
                left -= float(d[x])
                d = d.clone()
                d[x] = 0
        took.append(len(path) - 1)
        paths.append(path + [-1] * (width - len(path)))
        if greedy:
            nexts.append(target[a + path[-1]])
        else:
            cdf = torch.cumsum(r, 0)
            over = (cdf > u[a] * cdf[-1]).nonzero()
            nexts.append(int(over[0]) if len(over) else -1)
    return _ints(took), _ints(paths), _ints(nexts)


def _exact_keep(st):
    bs, pools = st["bs"], st["pools"]
    bt = st["bt"].tolist()
    for s, (c, k, a) in enumerate(zip(st["ctx"].tolist(), st["q_len"].tolist(),
                                      st["n_accepted"].tolist())):
        path = st["path"][s].tolist()
        for j in range(1, a + 1):
            p, q = c - k + path[j], c - k + j
            pools[:, bt[s][q // bs], :, :, q % bs] = pools[:, bt[s][p // bs], :, :, p % bs]
    return pools


def _exact_copy(st):
    for a, b in st["pairs"].tolist():
        st["pools"][:, b] = st["pools"][:, a].clone()
    return st["pools"]
