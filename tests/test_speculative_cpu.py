"""Speculative decoding without a GPU: argument errors of the C entry points,
draft-tree masks and step metadata, block tables of forks and rejected drafts,
and the 64-bit restatement the GPU tests compare against."""
from __future__ import annotations

import itertools

import numpy as np
import pytest
import torch

from oracle import speculative_ref as R
from tinybatch_b200 import _native as N
from tinybatch_b200 import ops
from tinybatch_b200.block_manager import BlockManager, OutOfBlocks
from tinybatch_b200.kv_cache import PagedKVCache
from tinybatch_b200.model import Qwen2Paged
from tinybatch_b200.runtime import StepMeta, tree_masks

P = 256     # stands for an aligned pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    if not N.lib_path().exists():
        from tinybatch_b200 import build
        build.build()
    return N.load()


def attention(lib, **kw):
    a = dict(q=P, ld_q=256, out=P, ld_out=256, rows=4, pool=P, blocks=8, hq=4, hkv=2, hd=64, bs=16, bt=P,
             bt_ld=4, bt_w=4, q_start=P, q_len=P, ctx=P, n=1, mask=P, mask_ld=1, words=1, max_q=4, max_ctx=0,
             total=0, stream=None)
    a.update(kw)
    return lib.tb_paged_attention_tree(*a.values())


@pytest.mark.parametrize("change,needle", [
    (dict(hq=5), "heads"), (dict(hkv=0), "heads"), (dict(hq=516, ld_q=33024, ld_out=33024), "GQA group"),
    (dict(hd=96), "head_dim"), (dict(bs=0), "block_size"), (dict(blocks=0), "num_blocks"),
    (dict(bt_w=0), "block table"), (dict(bt_ld=-1), "block table"), (dict(ld_q=252), "ld_q"),
    (dict(ld_out=128), "ld_out"), (dict(words=0), "words"), (dict(words=5, mask_ld=5), "words"),
    (dict(words=2), "words"), (dict(max_q=65), "max_q"), (dict(max_q=-1), "max_q"), (dict(n=-1), "n_seqs"),
    (dict(n=70000), "65535"), (dict(q=None), "null pointer"), (dict(mask=None), "null pointer"),
    (dict(ctx=None), "null pointer"), (dict(pool=P + 8), "aligned"), (dict(out=P + 2), "aligned"),
    (dict(mask=P + 4), "aligned")])
def test_attention_argument_errors(lib, change, needle):
    assert attention(lib, **change) == 1
    assert needle in lib.tb_last_error().decode()


@pytest.mark.parametrize("change", [dict(n=0), dict(max_q=0), dict(rows=0, max_q=0)])
def test_attention_of_nothing_launches_nothing(lib, change):
    assert attention(lib, q=None, **change) == 0


def verify(lib, **kw):
    a = dict(ids=P, parents=P, q_start=P, q_len=P, n=1, rows=4, max_q=4, probs=P, ld=100, vocab=100, draft=None,
             ld_d=0, n_d=0, d_rows=None, u=P, took=P, path=P, path_ld=4, path_w=4, nxt=P, stream=None)
    a.update(kw)
    return lib.tb_verify_drafts(*a.values())


@pytest.mark.parametrize("change,needle", [
    (dict(n=-1), "n_seqs"), (dict(rows=-1), "n_rows"), (dict(path_w=0), "path"), (dict(path_ld=3), "path"),
    (dict(max_q=257), "256 nodes"), (dict(ids=None), "null pointer"), (dict(nxt=None), "null pointer"),
    (dict(vocab=0), "vocab"), (dict(ld=99), "vocab"), (dict(probs=None), "probs"), (dict(u=None), "uniforms"),
    (dict(draft=P), "go together"), (dict(d_rows=P), "go together"),
    (dict(draft=P, d_rows=P, ld_d=99, n_d=1), "draft_probs"), (dict(draft=P, d_rows=P, ld_d=100, n_d=-1), "draft")])
def test_verify_argument_errors(lib, change, needle):
    assert verify(lib, **change) == 1
    assert needle in lib.tb_last_error().decode()


def test_verify_of_nothing_launches_nothing(lib):
    assert verify(lib, n=0, ids=None) == 0
    assert lib.tb_verify_drafts_greedy(None, None, None, None, 0, 0, 0, None, None, None, 1, 1, None, None) == 0
    assert lib.tb_verify_drafts_greedy(P, P, P, P, 1, 4, 4, None, P, P, 4, 4, P, None) == 1


def pools_h(*ptrs):
    import ctypes
    return (ctypes.c_void_p * len(ptrs))(*ptrs)


def test_cache_move_argument_errors(lib):
    def copy(pools, layers=1, blocks=4, hkv=2, bs=16, hd=64, pairs=P, n=1):
        return lib.tb_copy_kv_blocks(pools, layers, blocks, hkv, bs, hd, pairs, n, None)

    def keep(pools, layers=1, hd=64, bt_ld=4, bt_w=4, path_ld=4, path_w=4, path=P, n=1):
        return lib.tb_keep_kv_path(pools, layers, 4, 2, 16, hd, P, bt_ld, bt_w, P, P, path, path_ld, path_w, P, n,
                                   None)

    one = pools_h(P)
    for rc, needle in [(copy(one, blocks=0), "pool shape"), (copy(one, hd=12), "head_dim"),
                       (copy(None), "pools_h"), (copy(pools_h(P + 8)), "aligned"), (copy(pools_h(None)), "aligned"),
                       (copy(one, n=-1), "n_pairs"), (copy(one, pairs=None), "pairs"),
                       (copy(one, pairs=P + 4), "pairs")]:
        assert rc == 1
    for change, needle in [(dict(hd=12), "head_dim"), (dict(bt_w=0), "bt_ld"), (dict(path_w=0), "path"),
                           (dict(path_ld=3), "path"), (dict(path=None), "null pointer"), (dict(n=-1), "n_seqs")]:
        assert keep(one, **change) == 1
        assert needle in lib.tb_last_error().decode()
    assert copy(one, n=0) == 0 and copy(None, layers=0) == 0 and keep(one, n=0) == 0


@pytest.mark.parametrize("change,needle", [
    (dict(blocks=0), "pool shape"), (dict(hkv=0), "pool shape"), (dict(bs=0), "pool shape"), (dict(hd=12), "head_dim"),
    (dict(layers=-1), "pool shape"), (dict(pools=None), "pools_h"), (dict(pools=P + 8), "aligned"),
    (dict(pools=0), "aligned"), (dict(n=-1), "n_pairs"), (dict(pairs=None), "pairs"), (dict(pairs=P + 4), "pairs"),
    (dict(bs=1 << 20, hd=1 << 10), "1 GiB")])
def test_copy_refusals_name_their_reason(lib, change, needle):
    a = dict(pools=P, layers=1, blocks=4, hkv=2, bs=16, hd=64, pairs=P, n=1, stream=None)
    a.update(change)
    if a["pools"] is not None:
        a["pools"] = pools_h(a["pools"] or None)
    assert lib.tb_copy_kv_blocks(*a.values()) == 1
    assert needle in lib.tb_last_error().decode()


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        ops.KVPools(torch.zeros(1, 4, 2, 1, 16, 64, dtype=torch.bfloat16))
    t = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.verify_drafts_greedy(t, t, t, t, t, t, t[None], t)


def test_row_pitches_of_more_than_31_bits_are_refused():
    """They would wrap in the C entries' arguments (nothing is allocated: meta tensors)."""
    def rows(pitch):
        return torch.empty_strided((2, 4), (pitch, 1), dtype=torch.int32, device="meta")
    assert ops._mat("path", rows(2**31 - 1), torch.int32, 2, -1)[1:] == (2**31 - 1, 4)
    for pitch in (2**31, 2**32 + 8):
        with pytest.raises(ValueError, match="path"):
            ops._mat("path", rows(pitch), torch.int32, 2, -1)


def test_copy_blocks_checks_its_pairs_on_the_host():
    cache = PagedKVCache(1, 4, 16, 1, 64, device="cpu")
    cache.copy_blocks([])
    with pytest.raises(IndexError):
        cache.copy_blocks([(0, 4)])
    with pytest.raises(IndexError):
        cache.copy_blocks([(-1, 2)])
    with pytest.raises(ValueError):
        cache.copy_blocks([(0, 2), (1, 2)])
    with pytest.raises(ValueError):
        cache.copy_blocks([(0, 2), (2, 3)])


def test_cache_handle_follows_its_pools(monkeypatch):
    """The handle of the cache moves never keeps the address of storage that a pool
    has left, whether the tensor or what it holds was exchanged."""
    monkeypatch.setattr(ops, "_device", lambda t: -1)     # CPU tensors stand for the pools
    cache = PagedKVCache(3, 4, 16, 1, 64, device="cpu")

    def current():
        return list(cache.handle().addresses) == [p.data_ptr() for p in cache.pools]
    first = cache.handle()
    assert current() and cache.handle() is first
    old = cache.pools[1].data
    cache.pools[1].data = torch.ones_like(old)
    assert current() and cache.handle() is not first
    cache.pools[2].set_(torch.ones_like(old))
    assert current()
    cache.pools[0] = torch.zeros_like(old)
    assert current()
    cache.pools = cache.pools[:2]
    assert current()


def test_tree_masks():
    mask, depth = tree_masks([[-1, 0, 0, 1], [-1], []])
    assert mask.dtype == np.int64 and mask.tolist() == [[1], [3], [5], [11], [1]]
    assert depth.tolist() == [0, 1, 1, 2, 0]
    chain = [-1] + list(range(129))
    mask, depth = tree_masks([chain])
    assert mask.shape == (130, 3) and depth[-1] == 129
    assert mask[63].tolist() == [-1, 0, 0] and mask[64].tolist() == [-1, 1, 0] and mask[129].tolist() == [-1, -1, 3]
    assert tree_masks([])[0].shape == (0, 1)
    for bad in ([0], [-1, 1], [-1, -1], [-1, 0, 3], [-1, -2]):
        with pytest.raises(ValueError):
            tree_masks([bad])
    with pytest.raises(ValueError, match="256"):
        tree_masks([[-1] + [0] * 256])


def test_step_metadata_of_trees():
    """Nodes take consecutive slots behind the context whatever their positions;
    every node gets a logits row; no decode or prefill work remains."""
    parents = [[-1, 0, 0, 1], [-1, 0]]
    mask, depth = tree_masks(parents)
    md = StepMeta([5, 6, 7, 8, 9, 10], [20, 21, 21, 22, 3, 4], [(0, 4), (4, 6)], [[9, 2], [4]], [24, 5], 16, 2,
                  "cpu", pinned=False, all_logits=True, trees=mask)
    assert md.slots.tolist() == [36, 37, 38, 39, 67, 68]          # positions 20..23 of block 2, 3..4 of 4
    assert md.positions.tolist() == [20, 21, 21, 22, 3, 4] and md.ids.tolist() == [5, 6, 7, 8, 9, 10]
    assert md.row_dst.tolist() == list(range(6)) and md.n_out == 6
    assert md.n_dec == md.n_pre == 0 and md.n_tree == 2 and md.work.shape[0] == 0
    assert md.tree_mask.tolist() == mask.tolist() and md.tree_bt.tolist() == [[9, 2], [4, -1]]
    assert md.tree_q_start.tolist() == [0, 4] and md.tree_q_len.tolist() == [4, 2]
    assert md.tree_ctx.tolist() == [24, 5] and (md.tree_max_q, md.tree_max_ctx, md.tree_ctx_sum) == (4, 24, 29)
    with pytest.raises(IndexError):
        StepMeta([1, 2], [16, 17], [(0, 2)], [[3]], [18], 16, 2, "cpu", pinned=False, trees=mask[:2])
    with pytest.raises(ValueError):
        StepMeta([1, 2], [0, 1], [(0, 2)], [[3]], [2], 16, 2, "cpu", pinned=False, trees=mask[:1])


@pytest.mark.parametrize("ids,parents,tables,ctx,needle", [
    ([], [], [], [], "at least one tree"), ([1, 2], [[-1, 0, 0]], [[0]], [10], "3 nodes, 2 token ids"),
    ([1, 2, 3, 4], [[-1, 0, 0]], [[0]], [10], "3 nodes, 4 token ids"), ([1], [[-1]], [], [10], "per tree"),
    ([1], [[-1]], [[0]], [10, 11], "per tree"), ([1, 2], [[-1, 0]], [[0]], [1], "context holds"),
    ([1], [[-1], []], [[0], [1]], [10, 5], "has a root")])
def test_forward_tree_argument_errors(ids, parents, tables, ctx, needle):
    class OneRank:
        world = 1
    with pytest.raises(ValueError, match=needle):
        Qwen2Paged.forward_tree(OneRank(), ids, parents, tables, ctx, None)


def test_forward_tree_refuses_blocks_outside_the_pool():
    class OneRank:
        world = 1
    cache = PagedKVCache(1, 4, 16, 1, 64, device="cpu")
    for tables in ([[0, 4], [1]], [[0, 1], [2**30]]):
        with pytest.raises(IndexError, match="out of range"):
            Qwen2Paged.forward_tree(OneRank(), [5, 6], [[-1], [-1]], tables, [20, 3], cache)


def test_forward_tree_refuses_negative_blocks_inside_the_context():
    """A slot of a negative block wraps to another sequence's (-2^28 * 16 is slot 0 in 32
    bits); -1 may pad the table behind the context only."""
    class OneRank:
        world, device = 1, "cpu"

        class cfg:
            n_heads, n_kv_heads = 2, 1

        class dm:
            @staticmethod
            def forward(md, pools, sample):
                return None
    cache = PagedKVCache(1, 4, 16, 1, 64, device="cpu")
    for table in ([0, -1], [-1, 0], [-2**28, 0], [0, -2**28]):
        with pytest.raises(IndexError, match="out of range"):
            Qwen2Paged.forward_tree(OneRank(), [5], [[-1]], [table], [17], cache)
    md, _ = Qwen2Paged.forward_tree(OneRank(), [5, 6], [[-1], [-1]], [[3, -1], [0, 2]], [16, 17], cache)
    assert md.slots.tolist() == [63, 32] and md.tree_bt.tolist() == [[3, -1], [0, 2]]


def test_buffers_of_growing_batches_are_replaced_a_few_times_only():
    """Trees that grow a row a step: the retired sets, which stay for graphs over them, hold
    no more than the one in use."""
    from types import SimpleNamespace

    from tinybatch_b200.config import named_config
    from tinybatch_b200.runtime import DeviceModel
    dm = DeviceModel.__new__(DeviceModel)
    dm.cfg, dm.device = named_config("tiny"), "cpu"
    dm.w = SimpleNamespace(n_q=2, ff=dm.cfg.d_ff)
    dm._alloc(64, 16)
    for rows in range(1, 600):
        dm.ensure(rows, rows)
        assert dm.T_max >= rows and dm.logits.shape[0] >= rows and dm.h.shape[0] == dm.T_max
    assert dm._alloc_gen == 6                            # 32, 64, 128, 256, 512, 1024 rows of logits
    retired = sum(t[8].shape[0] for t in dm._retired)
    assert dm.logits.shape[0] == 1024 and retired <= 1024
    dm.ensure(5000, 20)
    assert (dm.T_max, dm.S_max) == (5000, 1024)          # a large batch gets what it needs


def test_fork_and_trim_tables():
    bm = BlockManager(8, 4, False)
    table, _ = bm.allocate_prompt(list(range(10)))                # 2 full blocks and half a third
    fork, copies = bm.fork_table(table, 10)
    assert fork[:2] == table[:2] and copies == [(table[2], fork[2])] and fork[2] not in table
    assert [bm.blocks[b].ref_count for b in table] == [2, 2, 1] and bm.blocks[fork[2]].ref_count == 1
    assert bm.blocks[fork[2]].token_ids == [8, 9]
    whole, copies = bm.fork_table(table, 8)
    assert whole == table[:2] and copies == [] and bm.blocks[table[0]].ref_count == 3
    bm.free_table(whole)
    # rejected drafts: blocks behind the kept tokens come back, shared ones stay with the other
    fork += [bm._own(bm._fresh_block(), []).block_id for _ in range(2)]
    assert bm.num_free() == 2
    bm.trim_table(fork, 10)
    assert len(fork) == 3 and bm.num_free() == 4
    bm.trim_table(fork, 8)
    bm.trim_table(fork, 8)
    assert fork == table[:2] and bm.num_free() == 5
    bm.trim_table(fork, 0)
    assert fork == [] and [bm.blocks[b].ref_count for b in table] == [1, 1, 1]
    bm.free_table(table)
    assert bm.num_free() == 8
    for bad in (-1, 1):
        with pytest.raises(ValueError):
            bm.fork_table([], bad)


def test_fork_without_a_free_block_changes_nothing():
    bm = BlockManager(2, 4, False)
    table, _ = bm.allocate_prompt(list(range(6)))
    with pytest.raises(OutOfBlocks):
        bm.fork_table(table, 6)
    assert [b.ref_count for b in bm.blocks] == [1, 1]


def test_fork_keeps_prefix_cached_blocks_cached():
    bm = BlockManager(4, 4, True)
    table, _ = bm.allocate_prompt(list(range(8)))
    fork, _ = bm.fork_table(table, 8)
    bm.free_table(table)
    assert bm.num_free() == 2
    bm.free_table(fork)
    assert bm.num_free() == 4 and bm.allocate_prompt(list(range(8)))[1] == 8


def test_trimmed_drafts_leave_the_prefix_cache():
    """Drafts that append_slot published are not found any more once they are
    trimmed: neither in the block that keeps accepted tokens (later tokens
    overwrite it) nor in a released one."""
    prompt, drafts = [1, 2, 3, 4, 5, 6], [70, 80, 90, 91, 92, 93, 94]
    for kept, cached in ((6, 4), (7, 4), (8, 8), (9, 8), (12, 12)):
        bm = BlockManager(8, 4, True)
        table, _ = bm.allocate_prompt(prompt)
        tokens = list(prompt)
        for t in drafts:
            bm.append_slot(table, tokens)
            tokens.append(t)
        assert len(table) == 4 and sum(b.prefix_hash is not None for b in bm.blocks) == 3
        bm.trim_table(table, kept)
        assert bm.num_free() == 8 - len(table) and not bm.evictable
        assert all(bm.blocks[b].prefix_hash in bm.cache for b in bm.cache.values())
        other, hit = bm.allocate_prompt(tokens)
        assert hit == cached and other[:cached // 4] == table[:cached // 4]
        assert not set(other[cached // 4:]) & set(table)
        # the accepted continuation is published under its own tokens
        bm.free_table(other)
        tokens = tokens[:kept] + [500 + i for i in range(9)]
        for n in range(kept, len(tokens)):
            bm.append_slot(table, tokens[:n])
        full = (len(tokens) - 1) // 4        # append_slot publishes a block when the next one opens
        assert bm.allocate_prompt(tokens)[1] == 4 * full


def test_room_for_drafts_is_published_once_accepted():
    """reserve / trim_table / publish over several steps: what other prompts find is
    always a prefix of accepted tokens, and every full block of them."""
    bm = BlockManager(32, 4, True)
    tokens = [1, 2, 3, 4, 5, 6]                       # the last one's K/V are written by the next forward
    table, _ = bm.allocate_prompt(tokens[:5])
    for step, took in enumerate((0, 3, 1, 0, 4, 4, 2)):
        drafts = [1000 * step + j for j in range(1, 6)]
        bm.reserve(table, len(tokens) + len(drafts))
        assert len(table) == bm.blocks_needed(len(tokens) + len(drafts))
        other, hit = bm.allocate_prompt(tokens + drafts)
        assert hit == (len(tokens) - 1) // 4 * 4      # no draft is found while it may be rejected
        assert not set(other[hit // 4:]) & set(table)
        bm.free_table(other)
        for bid in other[hit // 4:]:                  # (forget what this look published)
            if bm.blocks[bid].prefix_hash is not None:
                bm.evictable.pop(bid)
                bm._unpublish(bm.blocks[bid])
                bm.free_ids.append(bid)
        before = len(tokens)
        tokens += drafts[:took] + [1000 * step + 9]
        bm.trim_table(table, len(tokens) - 1)
        assert len(table) == bm.blocks_needed(len(tokens) - 1)
        bm.publish(table, tokens[:-1], before - 1)
        assert bm.blocks[table[0]].ref_count == 1
    other, hit = bm.allocate_prompt(tokens)
    assert hit == (len(tokens) - 1) // 4 * 4 and other[:hit // 4] == table[:hit // 4]
    with pytest.raises(ValueError):
        bm.publish(table, tokens + [0] * 4)
    # the next token by append_slot, in the room that trim_table left
    fresh = BlockManager(8, 4, True)
    table, _ = fresh.allocate_prompt([1, 2, 3])
    fresh.reserve(table, 9)
    fresh.trim_table(table, 4)
    assert fresh.append_slot(table, [1, 2, 3, 4]) and len(table) == 2
    assert fresh.allocate_prompt([1, 2, 3, 4])[1] == 4


def test_reserve_takes_all_blocks_or_none():
    bm = BlockManager(4, 4, True)
    old, _ = bm.allocate_prompt(list(range(8)))
    bm.free_table(old)                                # two cached blocks, evictable
    table, _ = bm.allocate_prompt([50])
    with pytest.raises(OutOfBlocks):
        bm.reserve(table, 17)
    assert len(table) == 1 and bm.num_free() == 3 and len(bm.cache) == 2
    bm.reserve(table, 1)
    bm.reserve(table, 0)
    assert len(table) == 1
    bm.reserve(table, 16)
    assert len(table) == len(set(table)) == 4 and bm.num_free() == 0 and not bm.cache
    bm.trim_table(table, 0)
    off = BlockManager(2, 4, False)
    table, _ = off.allocate_prompt([1, 2, 3, 4])
    off.publish(table, [1, 2, 3, 4])
    assert not off.cache


def test_trim_keeps_what_others_share():
    """Shared blocks stay published for their other tables; a trim that would leave the
    next token to a shared block changes nothing."""
    bm = BlockManager(8, 4, True)
    table, _ = bm.allocate_prompt(list(range(12)))
    other, hit = bm.allocate_prompt(list(range(12)))
    assert hit == 12 and other == table
    for tokens in (6, 11, -1):
        with pytest.raises(ValueError):
            bm.trim_table(other, tokens)
        assert other == table and [bm.blocks[b].ref_count for b in table] == [2, 2, 2]
    bm.trim_table(other, 4)
    assert other == table[:1] and [bm.blocks[b].ref_count for b in table] == [2, 1, 1]
    assert bm.allocate_prompt(list(range(12)))[1] == 12
    with pytest.raises(ValueError, match="negative"):
        bm.trim_table(other, -100)


def test_oracle_follows_the_target_exactly():
    """The restatement's acceptance and residual, integrated over the draft and the
    test's uniform number on a grid, give the target's distribution: two
    siblings drawn without replacement from q, first emitted token."""
    p = torch.tensor([.5, .2, .3], dtype=torch.float64)
    q = torch.tensor([.2, .5, .3], dtype=torch.float64)
    total = torch.zeros(3, dtype=torch.float64)
    grid = 40
    for a, b in itertools.permutations(range(3), 2):
        weight = float(q[a] * q[b] / (1 - q[a]))
        probs = torch.stack([p, p, p])
        for i, j in itertools.product(range(grid), range(grid)):
            for k in range(20):
                u = torch.tensor([(k + .5) / 20, (i + .5) / grid, (j + .5) / grid], dtype=torch.float64)
                took, path, nxt = R.verify([0, a, b], [-1, 0, 0], [0], [3], probs, u, 2, q[None],
                                           torch.zeros(3, dtype=torch.int32))
                tok = ([0, a, b][path[0][1]] if took[0] else nxt[0])
                total[tok] += weight / (grid * grid * 20)
                if took[0] and path[0][1] == 1:
                    total[tok] += weight * 19 / (grid * grid * 20)
                    break
    # midpoint grids misplace a threshold by at most half a cell: two tests, one sample
    assert bool(((total - p).abs() <= 2 * 0.5 / grid + 0.5 / 20).all()), total
