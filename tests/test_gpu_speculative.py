"""Speculative decoding on the B200: attention of draft trees over the paged
cache, verification, cache moves, each against a 64-bit restatement
(oracle/speculative_ref.py), and a run of them together through the model.

Tolerance of the attention: inputs are the same bf16 values on both sides.  The
output is rounded to bf16 once (at most 2^-8 relative) and the softmax weights
are rounded to bf16 before they meet V (each at most 2^-8 relative, so at most
2^-8 sum p |v|).  Scores are sums of up to 128 products in fp32; with |x| below
64 in base 2 their error stays below 128 * 2^-24 * 64 < 5e-4, the relative
error of a weight; the running sum and P V add a few 1e-5.  So
|out - ref| <= 2^-8 |ref| + (2^-8 + 1e-3) sum p |v|, elementwise.
"""
from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # collected on CPU-only hosts, never run there
    pytest.skip("needs a CUDA device", allow_module_level=True)

from oracle import speculative_ref as R  # noqa: E402
from tinybatch_b200 import _native, ops  # noqa: E402
from tinybatch_b200.runtime import tree_masks  # noqa: E402

DEV = "cuda"
BAD_INDEX = 103


@pytest.fixture(autouse=True)
def _status_clean():
    _native.status(clear=True)
    yield
    _native.raise_on_status("kernel")


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def starts(lens):
    return [sum(lens[:i]) for i in range(len(lens))]


def random_tree(rng, n, branch=4):
    kids, par = [0], [-1]
    for i in range(1, n):
        p = rng.choice([j for j in range(i) if kids[j] < branch])
        par.append(p)
        kids.append(0)
        kids[p] += 1
    return par


def word_masks(masks, words):
    """Python-int masks as the op's int64 words on the device."""
    m = np.array([[(x >> (64 * w)) & (2**64 - 1) for w in range(words)] for x in masks] or
                 np.zeros((0, words)), dtype=np.uint64)
    return torch.from_numpy(m.reshape(-1, words).view(np.int64)).to(DEV)


class Case:
    """A batch of draft trees over a random pool, and its 64-bit reference."""

    def __init__(self, hq, hkv, hd, bs, q_lens, prefix, seed=0, masks=None, poison=True):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.hq, self.hkv, self.hd, self.bs = hq, hkv, hd, bs
        self.q_lens, self.ctx = q_lens, [p + k for p, k in zip(prefix, q_lens)]
        self.q_start = starts(q_lens)
        self.words = max(1, -(-max(q_lens) // 64))
        self.parents = [random_tree(rng, k) if k else [] for k in q_lens]
        self.masks = masks
        if masks is None:
            self.masks = []
            for par in self.parents:
                m = []
                for i, p in enumerate(par):
                    m.append((m[p] if p >= 0 else 0) | 1 << i)
                self.masks += m
        nb = [-(-c // bs) for c in self.ctx]
        num_blocks = sum(nb) + 3
        ids = list(range(num_blocks))
        rng.shuffle(ids)
        self.tables, at = [], 0
        for k in nb:
            self.tables.append(ids[at:at + k])
            at += k
        self.pool = torch.randn(num_blocks, 2, hkv, bs, hd, generator=g).bfloat16()
        if poison:      # blocks of nobody, and the last blocks' places past the contexts
            self.pool[ids[at:]] = math.nan
            for t, c in zip(self.tables, self.ctx):
                if c % bs:
                    self.pool[t[-1], :, :, c % bs:] = math.nan
        self.q = torch.randn(sum(q_lens), hq * hd, generator=g).bfloat16()

    def device(self):
        width = max(1, max(map(len, self.tables)))
        bt = i32([t + [-1] * (width - len(t)) for t in self.tables])
        return dict(q=self.q.to(DEV), pool=self.pool.to(DEV), bt=bt, q_start=i32(self.q_start),
                    q_len=i32(self.q_lens), ctx=i32(self.ctx), mask=word_masks(self.masks, self.words))

    def run(self, d, out=None, **kw):
        out = torch.full_like(d["q"], math.nan) if out is None else out
        ops.paged_attention_tree(
            d["q"], out, d["pool"], n_q_heads=self.hq, n_kv_heads=self.hkv, head_dim=self.hd,
            block_size=self.bs, block_tables=d["bt"], q_start=d["q_start"], q_len=d["q_len"],
            ctx_len=d["ctx"], tree_mask=d["mask"], **kw)
        return out

    def check(self, out):
        ref, spread = R.tree_attention(self.q, self.pool, self.tables, self.q_start, self.q_lens,
                                       self.ctx, self.masks, self.hq, self.hkv, self.hd)
        compare(out, ref, spread)


def compare(out, ref, spread):
    out = out.double().cpu()
    assert torch.equal(out.isnan(), ref.isnan())
    tol = 2**-8 * ref.abs() + (2**-8 + 1e-3) * spread + 1e-30
    ok = (out - ref).abs() <= tol
    ok |= ref.isnan() | (out == ref)
    worst = ((out - ref).abs() / tol).nan_to_num(0).max()
    assert bool(ok.all()), f"{int((~ok).sum())} elements off, worst {float(worst):.2f} x tolerance"


HEADS = [(14, 2, 64, 16), (40, 8, 128, 16), (64, 8, 128, 32), (12, 1, 64, 16), (3, 3, 128, 16),
         (4, 2, 16, 4), (14, 2, 64, 8), (5, 1, 128, 48)]


@pytest.mark.parametrize("hq,hkv,hd,bs", HEADS)
@pytest.mark.parametrize("q_lens,prefix", [
    ([1], [0]), ([1], [1]), ([5], [200]), ([1, 3, 8, 2], [0, 15, 16, 63]),
    ([6, 0, 26, 17], [300, 40, 61, 130]), ([64, 33], [1, 500]), ([7, 1, 30], [1500, 2047, 700])])
def test_tree_attention(hq, hkv, hd, bs, q_lens, prefix):
    c = Case(hq, hkv, hd, bs, q_lens, prefix, seed=hq + len(q_lens))
    c.check(c.run(c.device(), max_q=max(q_lens), max_ctx=max(c.ctx), ctx_total=sum(c.ctx)))


@pytest.mark.parametrize("q_lens,prefix", [([65, 20], [100, 3]), ([128], [0]), ([200, 131], [77, 40]),
                                           ([256], [130])])
def test_tree_attention_many_words(q_lens, prefix):
    """Trees beyond one mask word, their keys in many tiles, default sizes."""
    c = Case(4, 2, 64, 16, q_lens, prefix, seed=5)
    c.check(c.run(c.device()))


def shares(c, max_ctx, ctx_total):
    """(CTAs that share a context, whether sequences start longest first) as the launch
    chooses them for nodes of one 128-row tile."""
    n = len(c.ctx)
    assert max(c.q_lens) * (c.hq // c.hkv) <= 128
    per = max(ctx_total * c.hkv // 296, 256)
    split = next(k for k in (8, 4, 2, 1) if max_ctx // per >= k or k == 1)
    return split, (1 < n <= 64 and split * c.hkv * n > 296 and 4 * max_ctx * n > 5 * ctx_total
                   and max_ctx // split >= 1024)


@pytest.mark.parametrize("hq,hkv,hd,bs", [(10, 2, 128, 16), (7, 1, 64, 32), (5, 1, 128, 8)])
@pytest.mark.parametrize("split", [1, 2, 8])
def test_tree_attention_many_tiles_a_cta(hq, hkv, hd, bs, split):
    """A CTA that walks far more than 16 key tiles: every window of eight tiles' block
    ids, every lap of the rings."""
    c = Case(hq, hkv, hd, bs, [9, 1, 5], [1100 * split + 700, 1089, 64 * 33 * split - 5], seed=20 + split)
    hints = dict(max_ctx=300 * split, ctx_total=300 * split if split == 1 else 300)
    assert shares(c, **hints)[0] == split and min(c.ctx[0], c.ctx[2]) / split > 17 * 64
    c.check(c.run(c.device(), max_q=9, **hints))


@pytest.mark.parametrize("n,hkv,longest,total,split", [
    (40, 8, 1100, 33000, 1),            # more sequences than lanes of a warp
    (64, 8, 1030, 50000, 1), (20, 16, 1500, 22500, 1), (10, 8, 8192, None, 4)])
@pytest.mark.parametrize("hd,bs", [(64, 16), (64, 8)])
def test_tree_attention_longest_sequences_first(n, hkv, longest, total, split, hd, bs):
    """Ragged batches whose CTAs take the sequences by length: ties, a sequence without
    nodes, and one whose bad length ranks first."""
    rng = random.Random(n)
    if total is None:
        prefix = [rng.choice([3500, 3700, 3700, 4300]) for _ in range(n)]
    else:
        prefix = [rng.choice([0, 33, 33, 200, rng.randint(1, 400)]) for _ in range(n)]
    at, none, bad = n // 2, 2, n - 2
    q_lens = [rng.randint(1, 3) for _ in range(n)]
    q_lens[none] = 0
    prefix[at] = longest - q_lens[at]
    c = Case(hkv, hkv, hd, bs, q_lens, prefix, seed=21)
    total = total or sum(c.ctx)
    assert shares(c, longest, total) == (split, True)
    d = c.device()
    good = c.run(d, max_q=3, max_ctx=longest, ctx_total=total)
    c.check(good)
    d["ctx"][bad] = 10**9
    out = c.run(d, max_q=3, max_ctx=longest, ctx_total=total)
    torch.cuda.synchronize()
    assert _native.status(clear=True) == BAD_INDEX
    lost = range(c.q_start[bad], c.q_start[bad] + q_lens[bad])
    rest = [i for i in range(sum(q_lens)) if i not in lost]
    assert torch.equal(out[rest], good[rest]) and bool(out[list(lost)].isnan().all())


@pytest.mark.parametrize("hints", [dict(), dict(max_ctx=1, ctx_total=1), dict(max_ctx=10**6, ctx_total=5),
                                   dict(max_ctx=5, ctx_total=10**12)])
def test_tree_attention_hints_only_share_out(hints):
    c = Case(10, 2, 128, 16, [9, 4, 1], [900, 20, 333], seed=6)
    c.check(c.run(c.device(), max_q=9, **hints))


@pytest.mark.parametrize("hq,hkv,hd,bs", [(10, 2, 128, 16), (14, 2, 64, 16), (4, 2, 16, 4)])
def test_tree_attention_arbitrary_masks(hq, hkv, hd, bs):
    """Masks that are no ancestor masks: later nodes, not the node itself, bits past
    the tree, nothing at all (with and without keys before the drafts)."""
    rng = random.Random(3)
    q_lens, prefix = [6, 40, 3], [0, 90, 0]
    masks = [rng.getrandbits(64) for _ in range(sum(q_lens))]
    masks[1] = masks[7] = masks[46] = 0
    masks[47] = ~0b111 & (2**64 - 1)          # only bits past its tree of three nodes
    c = Case(hq, hkv, hd, bs, q_lens, prefix, seed=7, masks=masks)
    out = c.run(c.device())
    c.check(out)
    assert float(out[1].abs().max()) == 0.0 and float(out[46].abs().max()) == 0.0
    assert float(out[47].abs().max()) == 0.0


@pytest.mark.parametrize("hq,hkv,hd,bs", [(10, 2, 128, 16), (14, 2, 64, 16), (4, 2, 16, 4)])
@pytest.mark.parametrize("prefix", [0, 50, 700])
def test_tree_attention_nonfinite_in_hidden_nodes(hq, hkv, hd, bs, prefix):
    """Infinities and NaN in the keys and values of a node reach the rows that see
    it and no others."""
    q_lens = [20]
    c = Case(hq, hkv, hd, bs, q_lens, [prefix], seed=8)
    leaf = [i for i in range(1, 20) if i not in c.parents[0]]
    for what, node, value in ((0, leaf[0], math.inf), (1, leaf[1], math.nan), (1, leaf[2], -math.inf),
                              (0, leaf[3], math.nan)):
        p = prefix + node
        c.pool[c.tables[0][p // bs], what, :, p % bs, 1::3] = value
    ref, spread = R.tree_attention(c.q, c.pool, c.tables, c.q_start, c.q_lens, c.ctx, c.masks, hq,
                                   hkv, hd)
    out = c.run(c.device()).double().cpu()
    touched = leaf[:4]
    clean = [i for i in range(20) if i not in touched]
    assert bool(ref[clean].isfinite().all())
    compare(out[clean], ref[clean], spread[clean])
    # values: the same columns are lost (a weight that underflows may turn inf to NaN)
    for i in (leaf[1], leaf[2]):
        assert torch.equal(out[i].isfinite(), ref[i].isfinite())
    assert bool(out[leaf[3]].isnan().all())


def test_tree_attention_strided_rows_and_untouched_rows():
    """q and out as slices of wider rows, a block table and a mask that are slices
    too, a batch whose sequences leave rows before, between and behind them."""
    hq, hkv, hd, bs = 10, 2, 64, 16
    c = Case(hq, hkv, hd, bs, [7, 5], [40, 120], seed=9)
    d = c.device()
    rows = [3 + i for i in range(7)] + [12 + i for i in range(5)]
    T = 20
    wide_q = torch.full((T, hq * hd + 64), math.nan, dtype=torch.bfloat16, device=DEV)
    wide_o = torch.full((T, hq * hd + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    wide_m = torch.full((T, 3), -1, dtype=torch.int64, device=DEV)
    wide_q[rows, 32:32 + hq * hd] = d["q"]
    wide_m[rows, 1] = d["mask"][:, 0]
    wide_t = torch.full((2, d["bt"].shape[1] + 9), 10**6, dtype=torch.int32, device=DEV)
    wide_t[:, 4:4 + d["bt"].shape[1]] = d["bt"]
    d.update(q=wide_q[:, 32:32 + hq * hd], mask=wide_m[:, 1:2], q_start=i32([3, 12]),
             bt=wide_t[:, 4:4 + d["bt"].shape[1]])
    c.run(d, out=wide_o[:, :hq * hd], max_q=7)
    c.check(wide_o[rows, :hq * hd])
    others = [i for i in range(T) if i not in rows]
    assert bool((wide_o[others] == 7.0).all()) and bool((wide_o[:, hq * hd:] == 7.0).all())


def test_tree_attention_in_place_and_on_a_side_stream():
    c = Case(40, 8, 128, 16, [25, 9], [2000, 70], seed=10)
    d = c.device()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = c.run(d, max_q=25)
        c.run(d, out=d["q"], max_q=25)
    torch.cuda.current_stream().wait_stream(s)
    c.check(want)
    assert torch.equal(want, d["q"])


def test_tree_attention_captured_twice_and_replayed_together():
    """Two graphs of the call share no workspace: replayed on two streams at once,
    one with new queries and lengths in place, both are right."""
    cases = [Case(40, 8, 128, 16, [12, 30], [900, 100], seed=11),
             Case(40, 8, 128, 16, [12, 30], [900, 100], seed=12)]
    ds = [c.device() for c in cases]
    outs = [torch.zeros_like(d["q"]) for d in ds]
    for c, d, o in zip(cases, ds, outs):
        c.run(d, out=o, max_q=30)
    torch.cuda.synchronize()
    graphs = []
    for c, d, o in zip(cases, ds, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run(d, out=o, max_q=30)
        graphs.append(g)
    # other queries, and other contexts (shorter, in the same blocks) for the second
    cases[1].q = Case(40, 8, 128, 16, [12, 30], [900, 100], seed=13).q
    cases[1].ctx = [700, 120]
    ds[1]["q"].copy_(cases[1].q)
    ds[1]["ctx"].copy_(i32(cases[1].ctx))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for o in outs:
        o.fill_(math.nan)
    torch.cuda.synchronize()
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        c.check(o)


def test_tree_attention_same_bits_twice():
    c = Case(64, 8, 128, 16, [40, 64, 7], [3000, 1000, 9], seed=14)
    d = c.device()
    a, b = c.run(d, max_ctx=3040, ctx_total=4120), c.run(d, max_ctx=3040, ctx_total=4120)
    assert torch.equal(a, b)
    c.check(a)


@pytest.mark.parametrize("hd,bs", [(64, 16), (16, 4)])
def test_tree_attention_bad_metadata_is_refused(hd, bs):
    """Sequences whose metadata leave the batch, the mask or the block table set
    the status word and write nothing; the others are computed."""
    c = Case(4, 2, hd, bs, [4, 4, 4, 4, 4], [30, 30, 30, 30, 30], seed=15)
    d = c.device()
    good = c.run(d)
    for name, at, value in (("q_start", 1, 17), ("q_start", 1, -1), ("q_len", 1, 21), ("q_len", 1, -1),
                            ("q_len", 1, 70), ("ctx", 1, 3), ("ctx", 1, 10**9), ("ctx", 1, -5)):
        bad = dict(d, **{name: d[name].clone()})
        bad[name][at] = value
        out = c.run(bad)
        torch.cuda.synchronize()
        assert _native.status(clear=True) == BAD_INDEX, (name, value)
        rest = [i for i in range(20) if not 4 <= i < 8]
        assert torch.equal(out[rest], good[rest]) and bool(out[4:8].isnan().all())
    bad = dict(d, bt=d["bt"].clone())
    bad["bt"][2, 0] = c.pool.shape[0]
    bad["bt"][3, 1] = -1
    out = c.run(bad)
    torch.cuda.synchronize()
    assert _native.status(clear=True) == BAD_INDEX
    assert torch.equal(out[:8], good[:8])


@pytest.mark.parametrize("hq,hkv,hd,bs", [(4, 2, 64, 16), (10, 2, 128, 8), (4, 2, 16, 4)])
def test_tree_attention_lengths_whose_difference_wraps_are_refused(hq, hkv, hd, bs):
    """ctx_len near -2^31: ctx_len - q_len leaves 32 bits and must not pass for a long prefix."""
    c = Case(hq, hkv, hd, bs, [4, 4, 4], [30, 30, 30], seed=15)
    d = c.device()
    good = c.run(d)
    rest = [0, 1, 2, 3, 8, 9, 10, 11]
    for value in (-2**31, -2**31 + 1, -2**31 + 3, -2**31 + 4):
        bad = dict(d, ctx=d["ctx"].clone())
        bad["ctx"][1] = value
        out = c.run(bad)
        torch.cuda.synchronize()
        assert _native.status(clear=True) == BAD_INDEX
        assert torch.equal(out[rest], good[rest]) and bool(out[4:8].isnan().all())


@pytest.mark.parametrize("hq,hkv,hd,bs", [(10, 2, 128, 16), (14, 2, 64, 16), (10, 2, 128, 8), (4, 2, 16, 4)])
@pytest.mark.parametrize("at", [0, -1])
def test_tree_attention_leaves_sequences_with_bad_blocks_out(hq, hkv, hd, bs, at):
    """A block id out of range, the first of a context or the last (nodes that few rows
    see): every row of the sequence stays as it was, whether one CTA or
    several share the context; the others' bits do not change."""
    c = Case(hq, hkv, hd, bs, [30, 30, 4], [600, 9, 40], seed=17)
    d = c.device()
    for split in (dict(max_ctx=630, ctx_total=630 + 39 + 44), dict(max_ctx=1, ctx_total=1)):
        good = c.run(d, **split)
        for seq in range(3):
            for value in (c.pool.shape[0], -1, 2**31 - 1, -2**31):
                bad = dict(d, bt=d["bt"].clone())
                bad["bt"][seq, at % len(c.tables[seq])] = value
                out = c.run(bad, **split)
                torch.cuda.synchronize()
                assert _native.status(clear=True) == BAD_INDEX
                lost = range(c.q_start[seq], c.q_start[seq] + c.q_lens[seq])
                rest = [i for i in range(64) if i not in lost]
                assert torch.equal(out[rest], good[rest]) and bool(out[list(lost)].isnan().all())


@pytest.mark.parametrize("hd,bs", [(64, 16), (16, 4)])
def test_tree_attention_max_q_zero(hd, bs):
    """max_q = 0 is right for a batch without nodes and reported for any other."""
    c = Case(4, 2, hd, bs, [4, 3], [30, 7], seed=18)
    d = c.device()
    out = c.run(d, max_q=0)
    torch.cuda.synchronize()
    assert _native.status(clear=True) == BAD_INDEX and bool(out.isnan().all())
    out = c.run(dict(d, q_len=i32([0, 0])), max_q=0)
    torch.cuda.synchronize()
    assert _native.status() == 0 and bool(out.isnan().all())


def test_tree_attention_refuses_arguments():
    c = Case(4, 2, 64, 16, [4], [30], seed=16)
    d = c.device()
    with pytest.raises(ValueError, match="q:"):
        c.run(dict(d, q=d["q"].float()))
    with pytest.raises(ValueError, match="tree_mask"):
        c.run(dict(d, mask=d["mask"].int()))
    with pytest.raises(ValueError, match="block_tables"):
        c.run(dict(d, bt=d["bt"].cpu()))
    with pytest.raises(ValueError, match="kv_pool"):
        c.run(dict(d, pool=d["pool"][..., :32]))
    with pytest.raises(ValueError, match="columns"):
        c.run(dict(d, q=d["q"][:, :192]))
    with pytest.raises(ValueError, match="contiguous"):
        c.run(dict(d, pool=d["pool"][::2]))
    with pytest.raises(_native.NativeError, match="max_q"):
        c.run(d, max_q=65)
    with pytest.raises(_native.NativeError, match="1 to 4 words"):
        c.run(dict(d, mask=torch.zeros(4, 5, dtype=torch.int64, device=DEV)))
    wide = torch.zeros(4, 4 * 64 + 4, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(_native.NativeError, match="multiples of 8"):
        c.run(dict(d, q=wide[:, :256]))
    with pytest.raises(_native.NativeError, match="aligned"):
        odd = torch.zeros(4 * 256 + 8, dtype=torch.bfloat16, device=DEV)[1:1025].view(4, 256)
        c.run(dict(d, q=odd))
    empty = {k: v[:0] if k in ("q", "mask", "bt", "q_start", "q_len", "ctx") else v for k, v in d.items()}
    assert c.run(empty).shape[0] == 0       # no sequences: nothing to do


# ------------------------------------------------------------- verification


def drafts(rng, n, nodes, vocab, branch=4, lens=None):
    lens = lens or [nodes if i == 0 else rng.randint(0, nodes) for i in range(n)]
    parents = [random_tree(rng, k, branch) if k else [] for k in lens]
    return lens, parents, [p for t in parents for p in t]


def outputs(n, width):
    return (torch.full((n,), 99, dtype=torch.int32, device=DEV),
            torch.full((n, width), 99, dtype=torch.int32, device=DEV),
            torch.full((n,), 99, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("n,nodes,vocab,width", [(1, 1, 5, 1), (1, 16, 3, 6), (7, 40, 4, 9), (130, 6, 2, 7),
                                                 (3, 256, 3, 256), (5, 30, 3, 2)])
def test_verify_greedy(n, nodes, vocab, width):
    rng = random.Random(n + nodes)
    lens, _, parents = drafts(rng, n, nodes, vocab)
    ids = [rng.randrange(vocab) for _ in parents]
    target = [rng.randrange(vocab) for _ in parents]
    took, path, nxt = outputs(n, width)
    ops.verify_drafts_greedy(i32(ids), i32(parents), i32(starts(lens)), i32(lens), i32(target), took,
                             path, nxt, max_q=nodes)
    want = R.verify_greedy(ids, parents, starts(lens), lens, target, width)
    assert (took.tolist(), path.tolist(), nxt.tolist()) == want


def distributions(g, rows, vocab, spread=2.0):
    return torch.softmax(torch.randn(rows, vocab, generator=g) * spread, -1)


def draw_children(rng, parents, q, rows):
    """Ids of every node: children of a node drawn from its row of q without
    replacement, in node order."""
    ids, taken = [0] * len(parents), {}
    for i, p in enumerate(parents):
        if p < 0:
            continue
        key = (rows[i], p)
        weights = q[rows[i]].tolist()
        for x in taken.get(key, []):
            weights[x] = 0.0
        if sum(weights) <= 0:
            weights = [1.0] * len(weights)
        ids[i] = rng.choices(range(len(weights)), weights)[0]
        taken.setdefault(key, []).append(ids[i])
    return ids


@pytest.mark.parametrize("n,nodes,vocab,branch,width", [
    (1, 1, 50, 1, 1), (6, 6, 20, 1, 6), (20, 12, 9, 4, 8), (9, 40, 1000, 4, 7), (4, 9, 4099, 3, 5),
    (3, 64, 30, 16, 10), (2, 30, 7, 30, 2), (5, 200, 300, 4, 12)])
@pytest.mark.parametrize("kind", ["drawn", "picked", "mixed"])
def test_verify_sampled(n, nodes, vocab, branch, width, kind):
    rng = random.Random(100 * n + nodes)
    g = torch.Generator().manual_seed(n + vocab)
    lens, trees, parents = drafts(rng, n, nodes, vocab, branch)
    T = len(parents)
    p = distributions(g, T, vocab)
    q = distributions(g, T, vocab)
    q = (0.6 * q + 0.4 * p).float()
    parent_row = [a + max(t, 0) for a, tree in zip(starts(lens), trees) for t in tree]
    ids = draw_children(rng, parents, q, parent_row)
    u = torch.rand(T, generator=g)
    rows = None
    if kind != "picked":
        rows = torch.arange(T, dtype=torch.int32)
        if kind == "mixed":
            rows[torch.rand(T, generator=g) < 0.4] = -1
    took, path, nxt = outputs(n, width)
    extra = {} if rows is None else dict(draft_probs=q.to(DEV), draft_rows=rows.to(DEV))
    ops.verify_drafts(i32(ids), i32(parents), i32(starts(lens)), i32(lens), p.to(DEV), u.to(DEV), took,
                      path, nxt, max_q=nodes, **extra)
    want = R.verify(ids, parents, starts(lens), lens, p, u, width, None if rows is None else q, rows)
    assert (took.tolist(), path.tolist(), nxt.tolist()) == want


@pytest.mark.parametrize("vocab,pad,shift", [(152064, 0, 0), (151936, 3, 0), (50257, 0, 1), (1, 0, 0),
                                             (127, 1, 2), (8191, 5, 3)])
def test_verify_sampled_wide_and_strided(vocab, pad, shift):
    """Full vocabularies, odd sizes, pitches and base addresses that are no multiple
    of 16 bytes."""
    rng = random.Random(vocab)
    g = torch.Generator().manual_seed(vocab)
    lens = [6, 4, 1, 9]
    lens, trees, parents = drafts(rng, 4, 9, vocab, 2, lens)
    T = len(parents)

    def place(x):
        flat = torch.zeros(T * (vocab + pad) + shift + 4)
        flat = flat.to(DEV)[shift:shift + T * (vocab + pad)].view(T, vocab + pad)[:, :vocab]
        flat.copy_(x)
        return flat

    p = distributions(g, T, vocab, 3.0)
    q = (0.5 * p + 0.5 * distributions(g, T, vocab, 3.0)).float()
    parent_row = [a + max(t, 0) for a, tree in zip(starts(lens), trees) for t in tree]
    ids = draw_children(rng, parents, q, parent_row)
    for seed in range(3):
        u = torch.rand(T, generator=torch.Generator().manual_seed(seed))
        took, path, nxt = outputs(4, 8)
        rows = torch.arange(T, dtype=torch.int32)
        ops.verify_drafts(i32(ids), i32(parents), i32(starts(lens)), i32(lens), place(p), u.to(DEV), took,
                          path, nxt, draft_probs=place(q), draft_rows=rows.to(DEV))
        assert (took.tolist(), path.tolist(), nxt.tolist()) == R.verify(
            ids, parents, starts(lens), lens, p, u, 8, q, rows)


@pytest.mark.parametrize("n,vocab", [
    (12, 152064), (10, 20011), (80, 152064), (160, 50257), (200, 152064), (300, 20000), (300, 152064),
    (9, 200003), (2, 163841), (1, 400000)])
@pytest.mark.parametrize("kind", ["drawn", "picked"])
def test_verify_sampled_serving_sizes(n, vocab, kind):
    """Real vocabularies in batches of every cluster size (8, 4, 2 and 1 CTAs a sequence
    from 10 sequences on): several batches of a segment, several steps of a batch; and few
    sequences whose vocabulary takes more than one step of 16 CTAs."""
    rng = random.Random(n + vocab)
    g = torch.Generator(device=DEV).manual_seed(n + vocab)
    nodes = 9 if n < 10 else 5 if n < 50 else 3
    lens = [nodes if i == 0 else rng.randint(0, nodes) for i in range(n)]
    parents = [p for k in lens for p in (random_tree(rng, k, 3) if k else [])]
    T = len(parents)
    p = torch.softmax(torch.randn(T, vocab, generator=g, device=DEV) * 3, -1)
    # a draft that often misses: siblings are reached, residuals sampled
    q = 0.6 * torch.softmax(torch.randn(T, vocab, generator=g, device=DEV) * 3, -1) + 0.4 * p
    parent_row = [a + max(x, 0) for a, k in zip(starts(lens), lens) for x in parents[a:a + k]]
    taken = {}
    ids = [0] * T
    for i, par in enumerate(parents):
        if par < 0:
            continue
        w = q[parent_row[i]].clone()
        w[taken.get(parent_row[i], [])] = 0
        ids[i] = int(torch.multinomial(w, 1, generator=g))
        taken.setdefault(parent_row[i], []).append(ids[i])
    u = torch.rand(T, generator=g, device=DEV)
    rows = torch.arange(T, dtype=torch.int32, device=DEV)
    took, path, nxt = outputs(n, 4)
    extra = dict(draft_probs=q, draft_rows=rows) if kind == "drawn" else {}
    ops.verify_drafts(i32(ids), i32(parents), i32(starts(lens)), i32(lens), p, u, took, path, nxt, max_q=nodes,
                      **extra)
    drawn = (q.cpu(), rows.cpu()) if kind == "drawn" else (None, None)
    want = R.verify(ids, parents, starts(lens), lens, p.cpu(), u.cpu(), 4, *drawn)
    assert (took.tolist(), path.tolist(), nxt.tolist()) == want


def test_verify_sampled_corners():
    """Point masses, draft rows that equal the target's, drafts of probability zero
    on either side, the same draft twice, u = 0, a target row without mass."""
    V = 8
    one = torch.eye(V)
    flat = torch.full((V,), 1 / V)
    half = torch.tensor([.5, .5, 0, 0, 0, 0, 0, 0])
    cases = [   # target after root, draft row, children, u of children, u of root
        (one[3], one[3], [3], [0.99], 0.5), (one[3], one[2], [2], [0.0], 0.5), (one[3], one[2], [2], [0.5], 0.0),
        (flat, flat, [1, 2, 3], [0.999999, 0.9999, 0.99], 0.3), (half, flat, [5, 0, 1], [0.0, 0.9, 0.4], 0.9),
        (flat, half, [5, 0, 1], [0.0, 0.3, 0.3], 0.7), (flat, half, [0, 0, 1, 1], [0.9, 0.0, 0.9, 0.0], 0.999),
        (torch.zeros(V), flat, [1, 2], [0.0, 0.5], 0.5), (0.5 * flat, flat, [1, 2, 1], [0.9, 0.95, 0.0], 0.1),
        (flat, one[4], [4, 5, 6], [0.9, 0.0, 0.0], 0.2), (half, half, [0, 1, 2], [0.999, 0.999, 0.0], 0.99)]
    for picked in (False, True):
        lens = [1 + len(c[2]) for c in cases]
        T = sum(lens)
        ids, parents, u, p, q = [], [], [], torch.zeros(T, V), torch.zeros(T, V)
        for target, draft, kids, uk, ur in cases:
            p[len(ids)], q[len(ids)] = target, draft
            for j in range(len(kids)):
                p[len(ids) + 1 + j] = flat
            ids += [0] + kids
            parents += [-1] + [0] * len(kids)
            u += [ur] + uk
        u = torch.tensor(u)
        rows = torch.arange(T, dtype=torch.int32)
        took, path, nxt = outputs(len(lens), 3)
        extra = {} if picked else dict(draft_probs=q.to(DEV), draft_rows=rows.to(DEV))
        ops.verify_drafts(i32(ids), i32(parents), i32(starts(lens)), i32(lens), p.to(DEV), u.to(DEV), took,
                          path, nxt, **extra)
        want = R.verify(ids, parents, starts(lens), lens, p, u, 3,
                        *((None, None) if picked else (q, rows)))
        assert (took.tolist(), path.tolist(), nxt.tolist()) == want


@pytest.mark.parametrize("kind", ["drawn", "picked"])
def test_verify_sampled_follows_the_target(kind):
    """The first emitted token of 60000 sequences with three drafts at the root is
    distributed as the target's row: every frequency within 5 standard
    deviations of a binomial count (V = 6 tokens)."""
    N, V = 60000, 6
    g = torch.Generator().manual_seed(4)
    p = torch.tensor([.35, .05, .2, .25, .05, .1])
    q = torch.tensor([.1, .3, .2, .05, .3, .05])
    if kind == "drawn":
        kids = torch.multinomial(q.expand(N, V), 3, generator=g)
    else:
        kids = torch.tensor([1, 3, 0]).expand(N, 3)
    ids = torch.cat([torch.zeros(N, 1, dtype=torch.long), kids], 1).int().view(-1).to(DEV)
    parents = i32([-1, 0, 0, 0]).repeat(N)
    lens, at = torch.full((N,), 4, dtype=torch.int32, device=DEV), torch.arange(0, 4 * N, 4, device=DEV).int()
    took, path, nxt = outputs(N, 2)
    extra = {}
    if kind == "drawn":
        extra = dict(draft_probs=q[None].to(DEV), draft_rows=torch.zeros(4 * N, dtype=torch.int32, device=DEV))
    ops.verify_drafts(ids, parents, at, lens, p.repeat(4 * N, 1).to(DEV),
                      torch.rand(4 * N, generator=g).to(DEV), took, path, nxt, **extra)
    first = torch.where(took > 0, ids.view(N, 4).gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], nxt)
    freq = torch.bincount(first.cpu(), minlength=V).double() / N
    sigma = (p.double() * (1 - p.double()) / N).sqrt()
    assert bool(((freq - p.double()).abs() <= 5 * sigma).all()), (freq, p)


def test_verify_bad_trees_are_refused():
    """Nodes with a parent that is no earlier node, an id outside the vocabulary or
    a draft row out of range are never accepted, sequences outside the batch
    give nothing; all set the status word."""
    V = 4
    p = torch.full((8, V), 1 / V, device=DEV)
    u = torch.zeros(8, device=DEV)
    ids = i32([0, 1, 2, 9, 0, 1, 2, 3])
    took, path, nxt = outputs(2, 4)

    def go(parents, q_start=(0, 4), q_len=(4, 4), the_ids=ids, **kw):
        for greedy in (False, True):
            if greedy and not kw:
                ops.verify_drafts_greedy(the_ids, i32(parents), i32(q_start), i32(q_len),
                                         i32([1, 2, 3, 0, 1, 2, 3, 0]), took, path, nxt)
            else:
                ops.verify_drafts(the_ids, i32(parents), i32(q_start), i32(q_len), p, u, took, path, nxt, **kw)
            torch.cuda.synchronize()
            yield _native.status(clear=True)

    assert BAD_INDEX in list(go([-1, 0, 1, 2, -1, 0, 1, 2]))         # id 9 in the sampled form
    fine = i32([0, 1, 2, 3, 0, 1, 2, 3])
    for status in go([-1, 5, 0, 0, -1, 0, 1, 2], the_ids=fine):
        assert status == BAD_INDEX and took.tolist()[1] == 3
    for status in go([-1, 0, 1, 2, -1, 0, 1, 2], q_start=(5, 4), the_ids=fine):
        assert status == BAD_INDEX and path.tolist()[0] == [-1] * 4 and nxt.tolist()[0] == -1
    for status in go([-1, 0, 1, 2, -1, 0, 1, 2], q_len=(-1, 4), the_ids=fine):
        assert status == BAD_INDEX and took.tolist() == [0, 3]
    for status in go([-1, 0, 1, 2, -1, 0, 1, 2], the_ids=fine, draft_probs=p[:2],
                     draft_rows=i32([2, -2, 0, 1, 0, 0, 0, 0])):
        assert status == BAD_INDEX


def test_verify_greedy_never_accepts_negative_ids():
    """A draft without an id does not match a node without a choice."""
    took, path, nxt = outputs(2, 3)
    ops.verify_drafts_greedy(i32([-1, -1, 4, -1, 4, 2]), i32([-1, 0, 0, -1, 0, 1]), i32([0, 3]), i32([3, 3]),
                             i32([-1, 3, 3, 4, 2, 7]), took, path, nxt)
    torch.cuda.synchronize()
    assert _native.status(clear=True) == BAD_INDEX
    assert took.tolist() == [0, 2] and nxt.tolist() == [-1, 7]      # (a root's id is not looked at)
    assert path.tolist() == [[0, -1, -1], [0, 1, 2]]


def test_verify_refuses_arguments():
    ids = i32([0, 1])
    p, u = torch.full((2, 3), 1 / 3, device=DEV), torch.zeros(2, device=DEV)
    base = (ids, i32([-1, 0]), i32([0]), i32([2]))
    took, path, nxt = outputs(1, 2)
    with pytest.raises(ValueError, match="probs"):
        ops.verify_drafts(*base, p.half(), u, took, path, nxt)
    with pytest.raises(ValueError, match="go together"):
        ops.verify_drafts(*base, p, u, took, path, nxt, draft_probs=p)
    with pytest.raises(ValueError, match="uniforms"):
        ops.verify_drafts(*base, p, u.double(), took, path, nxt)
    with pytest.raises(ValueError, match="path"):
        ops.verify_drafts(*base, p, u, took, path[0], nxt)
    with pytest.raises(ValueError, match="parents"):
        ops.verify_drafts_greedy(ids, base[1].long(), *base[2:], ids, took, path, nxt)
    with pytest.raises(_native.NativeError, match="256 nodes"):
        ops.verify_drafts(*base, p, u, took, path, nxt, max_q=257)
    with pytest.raises(_native.NativeError, match="probs"):
        ops.verify_drafts(*base, p[:1].expand(2, 3), u, took, path, nxt)
    ops.verify_drafts(ids[:0], ids[:0], ids[:0], ids[:0], p[:0], u[:0], took[:0], path[:0], nxt[:0])


def test_verify_without_any_draft_distribution():
    """draft_probs without rows: what None says, and a row that names one is reported."""
    p, u = torch.full((2, 3), 1 / 3, device=DEV), torch.tensor([0.5, 0.2], device=DEV)
    base = (i32([0, 1]), i32([-1, 0]), i32([0]), i32([2]), p, u)
    want = outputs(1, 2)
    ops.verify_drafts(*base, *want)
    for rows in ([-1, -1], [0, -1]):
        got = outputs(1, 2)
        ops.verify_drafts(*base, *got, draft_probs=p[:0], draft_rows=i32(rows))
        for a, b in zip(want, got):
            assert torch.equal(a, b)
        assert _native.status(clear=True) == (BAD_INDEX if rows[0] == 0 else 0)


def test_verify_of_sequences_without_any_row():
    """A padded batch that holds no tree: nothing accepted, nothing chosen."""
    none, zeros = torch.empty(0, dtype=torch.int32, device=DEV), i32([0, 0, 0])
    probs, u = torch.empty(0, 50, device=DEV), torch.empty(0, device=DEV)
    for call in (lambda *o: ops.verify_drafts_greedy(none, none, zeros, zeros, none, *o),
                 lambda *o: ops.verify_drafts(none, none, zeros, zeros, probs, u, *o),
                 lambda *o: ops.verify_drafts(none, none, zeros, zeros, probs, u, *o, draft_probs=probs,
                                              draft_rows=none)):
        took, path, nxt = outputs(3, 4)
        call(took, path, nxt)
        assert (took.tolist(), path.tolist(), nxt.tolist()) == ([0] * 3, [[-1] * 4] * 3, [-1] * 3)


def test_verify_captured_and_replayed():
    g = torch.Generator().manual_seed(1)
    p = distributions(g, 12, 5000).to(DEV)
    q = distributions(g, 12, 5000).to(DEV)
    ids, parents = torch.randint(0, 5000, (12,), generator=g).int().to(DEV), i32([-1, 0, 0, 1] * 3)
    u, rows = torch.rand(12, generator=g).to(DEV), i32(range(12))
    args = (ids, parents, i32([0, 4, 8]), i32([4, 4, 4]))
    took, path, nxt = outputs(3, 3)
    ops.verify_drafts(*args, p, u, took, path, nxt, draft_probs=q, draft_rows=rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.verify_drafts(*args, p, u, took, path, nxt, draft_probs=q, draft_rows=rows)
    for seed in range(4):
        u.copy_(torch.rand(12, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = R.verify(ids.tolist(), parents.tolist(), [0, 4, 8], [4, 4, 4], p.cpu(), u.cpu(), 3, q.cpu(),
                        rows.cpu())
        assert (took.tolist(), path.tolist(), nxt.tolist()) == want


# --------------------------------------------------------------- cache moves


def random_pools(layers, blocks, hkv, bs, hd, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(blocks, 2, hkv, bs, hd, generator=g).bfloat16() for _ in range(layers)]


@pytest.mark.parametrize("layers,hkv,bs,hd", [(1, 1, 1, 8), (3, 2, 16, 64), (5, 8, 16, 128), (2, 3, 4, 16),
                                              (130, 1, 4, 8), (2, 1, 48, 40)])
@pytest.mark.parametrize("stacked", [False, True])
def test_copy_blocks(layers, hkv, bs, hd, stacked):
    host = random_pools(layers, 12, hkv, bs, hd)
    pairs = [(0, 5), (0, 6), (11, 7), (3, 3), (2, 10)]
    dev = [p.to(DEV) for p in host]
    if stacked:
        dev = torch.stack(dev)
    ops.copy_kv_blocks(dev, i32(pairs))
    for p, d in zip(host, dev):
        want = p.clone()
        for a, b in pairs:
            want[b] = p[a]
        assert torch.equal(want, d.cpu())


def test_copy_blocks_many_pairs():
    host = random_pools(2, 1400, 2, 4, 64)
    order = torch.randperm(1400, generator=torch.Generator().manual_seed(2)).tolist()
    pairs = list(zip(order[:650], order[700:1350]))
    dev = [p.to(DEV) for p in host]
    ops.copy_kv_blocks(ops.KVPools(dev), i32(pairs))
    for p, d in zip(host, dev):
        want = p.clone()
        want[[b for _, b in pairs]] = p[[a for a, _ in pairs]]
        assert torch.equal(want, d.cpu())


@pytest.mark.parametrize("pairs,made", [
    ([(0, 1), (2, 3), (1, 4)], [(2, 3), (1, 4)]),       # 1 is written and read
    ([(0, 5), (2, 5), (3, 4)], [(3, 4)]),               # 5 is written twice
    ([(0, 12), (-1, 5), (2, 3)], [(2, 3)]), ([(12, 1), (2, -1)], []),
    ([(3, 3), (0, 3)], [])])                            # onto itself, and written by another
def test_copy_blocks_refuses_clashes(pairs, made):
    host = random_pools(2, 12, 2, 16, 64)
    dev = [p.to(DEV) for p in host]
    ops.copy_kv_blocks(dev, i32(pairs))
    torch.cuda.synchronize()
    assert _native.status(clear=True) == BAD_INDEX
    for p, d in zip(host, dev):
        want = p.clone()
        for a, b in made:
            want[b] = p[a]
        assert torch.equal(want, d.cpu())


def test_cache_moves_refuse_arguments():
    pools = [p.to(DEV) for p in random_pools(2, 4, 2, 16, 64)]
    with pytest.raises(ValueError, match="twice"):
        ops.copy_kv_blocks([pools[0], pools[0]], i32([(0, 1)]))
    with pytest.raises(ValueError, match="one shape"):
        ops.copy_kv_blocks([pools[0], pools[1][:2]], i32([(0, 1)]))
    with pytest.raises(ValueError, match="one shape"):
        ops.copy_kv_blocks([pools[0], pools[1].float()], i32([(0, 1)]))
    with pytest.raises(ValueError, match="pairs"):
        ops.copy_kv_blocks(pools, i32([(0, 1)]).long())
    with pytest.raises(ValueError, match="overlap"):
        ops.copy_kv_blocks(pools[0].expand(3, *pools[0].shape), i32([(0, 1)]))
    with pytest.raises(ValueError, match="CUDA"):
        ops.copy_kv_blocks([p.cpu() for p in pools], i32([(0, 1)]))
    ops.copy_kv_blocks(pools, i32([]).view(0, 2))


@pytest.mark.parametrize("layers,hkv,bs,hd", [(1, 1, 1, 8), (3, 2, 16, 64), (2, 8, 16, 128), (131, 1, 4, 16),
                                              (2, 40, 16, 128), (2, 3, 48, 40)])
@pytest.mark.parametrize("stacked", [False, True])
def test_keep_path(layers, hkv, bs, hd, stacked):
    rng = random.Random(hd)
    q_lens = [1, 9, 30, 0, 12, 25]
    ctx = [20, 9, 61, 7, 50, 33]
    took = [0, 8, 5, 0, 11, 1]
    paths = [[0] + sorted(rng.sample(range(1, k), t)) + [-1] * (13 - 1 - t) if k else [-1] * 13
             for k, t in zip(q_lens, took)]
    paths[1][:9] = list(range(9))                        # nothing moves
    need = [-(-c // bs) for c in ctx]
    ids = list(range(sum(need) + 2))
    rng.shuffle(ids)
    tables, at = [], 0
    for k in need:
        tables.append(ids[at:at + k])
        at += k
    host = random_pools(layers, len(ids), hkv, bs, hd)
    dev = [p.to(DEV) for p in host]
    if stacked:
        dev = torch.stack(dev)
    width = max(need)
    ops.keep_kv_path(dev, block_tables=i32([t + [-1] * (width - len(t)) for t in tables]), q_len=i32(q_lens),
                     ctx_len=i32(ctx), path=i32(paths), n_accepted=i32(took))
    for want, d in zip(R.keep_path(host, tables, q_lens, ctx, paths, took), dev):
        assert torch.equal(want, d.cpu())


@pytest.mark.parametrize("bs", [1, 4, 16])
def test_keep_path_partly_in_place(bs):
    """Paths whose first nodes, or all of them, stay where they are."""
    paths = [[0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 6], [0, 1, 2, 5, 7, -1], [0, 1, -1, -1, -1, -1],
             [0, 2, -1, -1, -1, -1]]
    took, q_lens, ctx = [5, 5, 4, 1, 1], [8] * 5, [8, 21, 33, 40, 11]
    need = [-(-c // bs) for c in ctx]
    ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(bs)).tolist()
    tables = [ids[sum(need[:i]):sum(need[:i + 1])] for i in range(5)]
    host = random_pools(3, len(ids), 2, bs, 64)
    dev = [p.to(DEV) for p in host]
    ops.keep_kv_path(dev, block_tables=i32([t + [-1] * (max(need) - len(t)) for t in tables]), q_len=i32(q_lens),
                     ctx_len=i32(ctx), path=i32(paths), n_accepted=i32(took))
    for want, d in zip(R.keep_path(host, tables, q_lens, ctx, paths, took), dev):
        assert torch.equal(want, d.cpu())


def test_keep_path_long_paths():
    """More accepted nodes than one batch of loads, chains shifted by one."""
    host = random_pools(2, 40, 2, 16, 64)
    k, c = 200, 230
    table = torch.randperm(40, generator=torch.Generator().manual_seed(0))[:15].tolist()
    path = [0] + list(range(2, 200))
    dev = [p.to(DEV) for p in host]
    ops.keep_kv_path(dev, block_tables=i32([table]), q_len=i32([k]), ctx_len=i32([c]), path=i32([path]),
                     n_accepted=i32([198]))
    for want, d in zip(R.keep_path(host, [table], [k], [c], [path], [198]), dev):
        assert torch.equal(want, d.cpu())


@pytest.mark.parametrize("change", [
    dict(path=[0, 2, 2, 5]), dict(path=[0, 3, 2, 5]), dict(path=[0, 0, 2, 5]), dict(path=[0, 1, 2, 6]),
    dict(path=[0, -1, 2, 5]), dict(took=4), dict(took=-1), dict(ctx=2), dict(ctx=10**9), dict(ctx=-3),
    dict(table=[99, 1]), dict(table=[0, -1]), dict(q_len=257), dict(q_len=3)])
def test_keep_path_bad_sequences_move_nothing(change):
    host = random_pools(2, 8, 2, 16, 64)
    dev = [p.to(DEV) for p in host]
    c = dict(dict(path=[0, 1, 3, 5], took=3, ctx=20, table=[4, 2], q_len=6), **change)
    good = dict(path=[0, 2, 4, -1], took=2, ctx=18, table=[5, 6], q_len=5)
    both = [c, good]
    ops.keep_kv_path(dev, block_tables=i32([x["table"] for x in both]), q_len=i32([x["q_len"] for x in both]),
                     ctx_len=i32([x["ctx"] for x in both]), path=i32([x["path"] for x in both]),
                     n_accepted=i32([x["took"] for x in both]))
    torch.cuda.synchronize()
    assert _native.status(clear=True) == BAD_INDEX
    for want, d in zip(R.keep_path(host, [good["table"]], [5], [18], [good["path"]], [2]), dev):
        assert torch.equal(want, d.cpu())


@pytest.mark.parametrize("ctx", [-2**31, -2**31 + 3, -2**31 + 5, 5])
def test_keep_path_lengths_whose_difference_wraps_move_nothing(ctx):
    """ctx_len - q_len must not pass for a position after leaving 32 bits."""
    host = random_pools(2, 8, 2, 16, 64)
    dev = [p.to(DEV) for p in host]
    ops.keep_kv_path(dev, block_tables=i32([[4, 2], [5, 6]]), q_len=i32([6, 5]), ctx_len=i32([ctx, 18]),
                     path=i32([[0, 1, 3, 5], [0, 2, 4, -1]]), n_accepted=i32([3, 2]))
    torch.cuda.synchronize()
    assert _native.status(clear=True) == BAD_INDEX
    for want, d in zip(R.keep_path(host, [[5, 6]], [5], [18], [[0, 2, 4, -1]], [2]), dev):
        assert torch.equal(want, d.cpu())


@pytest.mark.parametrize("q_start,ctx", [(-1, -1), (10**6, 10**6), (-2**31, -2**31), (2**31 - 1, 2**31 - 1)])
def test_sequences_without_nodes_take_part_in_nothing(q_start, ctx):
    """A padding row of the batch may hold anything beside its q_len of 0."""
    for hd, bs in ((64, 16), (16, 4)):
        c = Case(4, 2, hd, bs, [4, 0, 3], [30, 5, 7], seed=19)
        d = c.device()
        d["q_start"][1], d["ctx"][1], d["bt"][1] = q_start, ctx, -7
        c.check(c.run(d, max_q=4))
    ids, parents, lens, at = i32([0, 1, 2, 0, 1]), i32([-1, 0, 1, -1, 0]), i32([3, 0, 2]), i32([0, q_start, 3])
    p, u = torch.eye(3, device=DEV)[[1, 2, 0, 1, 2]].contiguous(), torch.full((5,), 0.5, device=DEV)
    for verify in (lambda *o: ops.verify_drafts(ids, parents, at, lens, p, u, *o),
                   lambda *o: ops.verify_drafts_greedy(ids, parents, at, lens, i32([1, 2, 0, 1, 2]), *o)):
        took, path, nxt = outputs(3, 3)
        verify(took, path, nxt)
        assert took.tolist() == [2, 0, 1] and nxt.tolist() == [0, -1, 2]
        assert path.tolist() == [[0, 1, 2], [-1, -1, -1], [0, 1, -1]]
    dev = [p.to(DEV) for p in random_pools(2, 4, 2, 16, 64)]
    before = [d.clone() for d in dev]
    ops.keep_kv_path(dev, block_tables=i32([[0], [99], [1]]), q_len=lens, ctx_len=i32([9, ctx, 9]), path=path,
                     n_accepted=i32([2, 0, 1]))
    assert all(torch.equal(a, b) for a, b in zip(dev, before))


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("name", ["tiny", "mid"])
def test_speculative_greedy_decoding_equals_plain_decoding(name):
    """A model decodes with draft trees (the forward over the tree, greedy
    verification, keeping the accepted path, trimming and forking tables) and
    emits the tokens that plain one-token steps emit, in fewer steps.  The
    drafts hold the plain run's continuation among wrong branches."""
    from tinybatch_b200 import weights
    from tinybatch_b200.block_manager import BlockManager
    from tinybatch_b200.config import named_config
    from tinybatch_b200.model import Qwen2Paged
    cfg = named_config("tiny") if name == "tiny" else named_config(
        "tiny", d_model=512, n_heads=8, n_kv_heads=2, head_dim=64, d_ff=768)
    model = Qwen2Paged.from_weights(cfg, weights.synthetic_weights(cfg, seed=0), DEV)
    bs, steps = 16, 24
    # two layers of six bf16 roundings (2^-8 each) between the two batch shapes' logits
    noise, compared = 2 * 6 * 2**-8, 0
    prompts = [list(range(3, 40)), list(range(90, 106)), [5]]

    def prefill(bm, cache):
        tables, seqs = [], []
        for p in prompts:
            table, _ = bm.allocate_prompt(p)
            seqs.append(list(p))
            tables.append(table)
        ends = np.cumsum([len(p) for p in prompts]).tolist()
        logits = model.forward([t for p in prompts for t in p], [i for p in prompts for i in range(len(p))],
                               [(e - len(p), e) for e, p in zip(ends, prompts)], tables,
                               [len(p) for p in prompts], cache)
        for s, t in zip(seqs, logits.argmax(-1).tolist()):
            s.append(t)
        return tables, seqs

    def room(bm, table, tokens):
        while len(table) * bs < tokens:
            table.append(bm._own(bm._fresh_block(), []).block_id)

    # plain: one token a step, through the same forward (a tree of one node)
    bm, cache = BlockManager(64, bs, False), model.make_kv_cache(64, bs)
    tables, plain = prefill(bm, cache)
    plain_logits = {}           # (sequence, tokens before) -> logits of the next token
    for _ in range(steps + 8):
        for t, s in zip(tables, plain):
            room(bm, t, len(s))
        md, logits = model.forward_tree([s[-1] for s in plain], [[-1]] * 3, tables, [len(s) for s in plain], cache)
        for i, (s, row) in enumerate(zip(plain, logits.cpu())):
            plain_logits[i, len(s)] = row
            s.append(int(row.argmax()))

    # speculative: chains of the plain continuation, some corrupted, among wrong siblings
    rng = random.Random(0)
    bm, cache = BlockManager(64, bs, False), model.make_kv_cache(64, bs)
    tables, spec = prefill(bm, cache)
    # a fork decodes beside its parent from a copy of the last block
    fork, copies = bm.fork_table(tables[0], len(prompts[0]))
    cache.copy_blocks(copies)
    assert copies and fork[:-1] == tables[0][:2]
    tables.append(fork)
    spec.append(list(spec[0]))
    want = plain + [plain[0]]
    forwards = 0
    while min(map(len, spec)) < min(len(p) for p in prompts) + steps:
        ids, parents = [], []
        for s, w in zip(spec, want):
            node_ids, par = [s[-1]], [-1]
            at, ahead = 0, w[len(s):len(s) + rng.randint(1, 5)]
            for k, tok in enumerate(ahead):
                for wrong in range(rng.randint(0, 2)):
                    node_ids.append((tok + 1 + wrong) % cfg.vocab_size)
                    par.append(at)
                node_ids.append(tok if rng.random() < 0.85 else (tok + 7) % cfg.vocab_size)
                par.append(at)
                at = len(par) - 1
            ids.append(node_ids)
            parents.append(par)
        ctx = [len(s) - 1 + len(n) for s, n in zip(spec, ids)]
        for t, c in zip(tables, ctx):
            room(bm, t, c)
        flat = [t for n in ids for t in n]
        md, target = model.forward_tree(flat, parents, tables, ctx, cache, sample=True)
        n = len(spec)
        took, path, nxt = outputs(n, 8)
        ops.verify_drafts_greedy(md.ids, i32([p for t in parents for p in t]), md.tree_q_start, md.tree_q_len,
                                 target, took, path, nxt, max_q=md.tree_max_q)
        cache.keep_path(block_tables=md.tree_bt, q_len=md.tree_q_len, ctx_len=md.tree_ctx, path=path,
                        n_accepted=took)
        forwards += 1
        logits = model.dm.logits[:md.T].cpu()
        for i, (s, a, pth) in enumerate(zip(spec, took.tolist(), path.tolist())):
            for k in range(a + 1):
                now = s + [ids[i][j] for j in pth[1:k + 1]]
                row = plain_logits.get((i % 3, len(now)))
                if row is not None and now == want[i][:len(now)]:
                    got = logits[starts([len(x) for x in ids])[i] + pth[k]]
                    assert float((got - row).abs().max()) <= noise * float(row.abs().max())
                    compared += 1
        for s, t, node_ids, a, pth, nx in zip(spec, tables, ids, took.tolist(), path.tolist(), nxt.tolist()):
            s += [node_ids[j] for j in pth[1:a + 1]] + [nx]
            bm.trim_table(t, len(s) - 1)
    # the plain run's tokens, up to a step whose two best logits the noise may swap
    for i, (s, w) in enumerate(zip(spec, want)):
        k = next((k for k, (x, y) in enumerate(zip(s, w)) if x != y), None)
        if k is not None:
            row = plain_logits[i % 3, k]
            assert float(row.max() - row[s[k]]) <= 2 * noise * float(row.abs().max())
    assert compared > 2 * steps
    assert forwards < steps
    for t in tables:
        bm.free_table(t)
    assert bm.num_free() == 64


def small_model(name):
    from tinybatch_b200 import weights
    from tinybatch_b200.config import named_config
    from tinybatch_b200.model import Qwen2Paged
    cfg = named_config("tiny") if name == "tiny" else named_config(
        "tiny", d_model=512, n_heads=8, n_kv_heads=2, head_dim=64, d_ff=768)
    return Qwen2Paged.from_weights(cfg, weights.synthetic_weights(cfg, seed=0), DEV)


# logits of one token in two batch shapes: two layers of six bf16 roundings (2^-8 each)
NOISE = 2 * 6 * 2**-8


def plain_logits(model, tokens, bs=16):
    """Logits after ``tokens`` from a prefill of all of them in a cache of its own."""
    blocks = -(-len(tokens) // bs)
    return model.forward(tokens, list(range(len(tokens))), [(0, len(tokens))], [list(range(blocks))], [len(tokens)],
                         model.make_kv_cache(blocks, bs))[0]


@pytest.mark.parametrize("name", ["tiny", "mid"])
def test_forward_tree_equals_the_plain_forward(name):
    """Every node's logits are those of a causal forward over the prompt and the
    node's path: positions, masks and slots, for branches, chains and a lone root."""
    model = small_model(name)
    V, bs = model.cfg.vocab_size, 16
    rng = random.Random(1)
    prompts = [[rng.randrange(V) for _ in range(k)] for k in (37, 16, 1, 90)]
    parents = [random_tree(rng, 12, 3), [-1] + list(range(6)), [-1, 0, 0, 0], [-1]]
    ids = [[rng.randrange(V) for _ in par] for par in parents]
    ctx = [len(p) + len(t) for p, t in zip(prompts, parents)]
    need = [-(-c // bs) for c in ctx]
    order = list(range(sum(need)))
    rng.shuffle(order)
    tables = [order[a:a + k] for a, k in zip(starts(need), need)]
    cache = model.make_kv_cache(sum(need), bs)
    ends = np.cumsum([len(p) for p in prompts]).tolist()
    model.forward([t for p in prompts for t in p], [i for p in prompts for i in range(len(p))],
                  [(e - len(p), e) for e, p in zip(ends, prompts)], tables, [len(p) for p in prompts], cache)
    md, logits = model.forward_tree([t for n in ids for t in n], parents, tables, ctx, cache)
    logits, positions, r0 = logits.clone(), md.positions.tolist(), 0
    for prompt, par, node_ids in zip(prompts, parents, ids):
        for i in range(len(par)):
            path, j = [], i
            while j >= 0:
                path.append(node_ids[j])
                j = par[j]
            # (a rotary position off by one would move the logits by less than the tolerance)
            assert positions[r0 + i] == len(prompt) + len(path) - 1
            want = plain_logits(model, prompt + path[::-1])
            assert float((logits[r0 + i] - want).abs().max()) <= NOISE * float(want.abs().max()), (r0, i)
        r0 += len(par)


def test_accepted_drafts_in_the_prefix_cache_hold_their_keys_and_values():
    """Steps of drafts in room from BlockManager.reserve, trimmed and published with the
    prefix cache on: a later prompt that finds the blocks computes only its tail,
    and its logits are those of a prefill of everything."""
    from tinybatch_b200.block_manager import BlockManager
    model = small_model("tiny")
    V, bs = model.cfg.vocab_size, 16
    rng = random.Random(2)
    bm, cache = BlockManager(64, bs), model.make_kv_cache(64, bs)
    seqs = [[rng.randrange(V) for _ in range(k)] for k in (20, 5)]
    tables = [bm.allocate_prompt(s)[0] for s in seqs]
    ends = np.cumsum([len(s) for s in seqs]).tolist()
    logits = model.forward([t for s in seqs for t in s], [i for s in seqs for i in range(len(s))],
                           [(e - len(s), e) for e, s in zip(ends, seqs)], tables, [len(s) for s in seqs], cache)
    for s, t in zip(seqs, logits.argmax(-1).tolist()):
        s.append(t)
    moved = 0
    for step in range(12):
        ids, parents = [], []
        for s in seqs:
            # right tokens (from a plain forward) in a chain, each behind a wrong sibling
            node_ids, par, at, ahead = [s[-1]], [-1], 0, list(s)
            for k in range(rng.randint(1, 4)):
                right = int(plain_logits(model, ahead).argmax())
                ahead.append(right)
                node_ids += [(right + 1) % V, right if rng.random() < 0.9 else (right + 2) % V]
                par += [at, at]
                at = len(par) - 1
            ids.append(node_ids)
            parents.append(par)
        ctx = [len(s) - 1 + len(n) for s, n in zip(seqs, ids)]
        for t, c in zip(tables, ctx):
            bm.reserve(t, c)
        md, target = model.forward_tree([t for n in ids for t in n], parents, tables, ctx, cache, sample=True)
        took, path, nxt = outputs(2, 6)
        ops.verify_drafts_greedy(md.ids, i32([p for t in parents for p in t]), md.tree_q_start, md.tree_q_len, target,
                                 took, path, nxt, max_q=md.tree_max_q)
        cache.keep_path(block_tables=md.tree_bt, q_len=md.tree_q_len, ctx_len=md.tree_ctx, path=path, n_accepted=took)
        for s, t, node_ids, a, pth, nx in zip(seqs, tables, ids, took.tolist(), path.tolist(), nxt.tolist()):
            before = len(s)
            s += [node_ids[j] for j in pth[1:a + 1]] + [nx]
            moved += a
            bm.trim_table(t, len(s) - 1)
            bm.publish(t, s[:-1], before - 1)
    assert moved > 12
    for s, t in zip(seqs, tables):
        prompt = s + [7, 8, 9]
        table, cached = bm.allocate_prompt(prompt)
        assert cached == (len(s) - 1) // bs * bs >= bs and table[:cached // bs] == t[:cached // bs]
        got = model.forward(prompt[cached:], list(range(cached, len(prompt))), [(0, len(prompt) - cached)], [table],
                            [len(prompt)], cache)[0]
        want = plain_logits(model, prompt)
        assert float((got - want).abs().max()) <= NOISE * float(want.abs().max())
