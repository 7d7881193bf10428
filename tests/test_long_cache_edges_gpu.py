"""The calls for long caches where their plans change: tables far wider than
the sequences (a program that captures a step gives its capacity), prompts among
single tokens, numbers of blocks and lengths of lists at which a choice leaves
its registers.  Each against the 64-bit forms and tolerances of its own tests."""
from __future__ import annotations

import numpy as np
import pytest

from test_attention_weights_gpu import Weigh
from test_block_attention_gpu import BlockCall
from test_keep_gpu import Evict
from test_tree_attention_gpu import TreeCall

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def widen(c, times, tokens=None):
    """The call's batch with a table `times` as wide, its other entries no pages."""
    pool = c.pool
    table = np.full((len(pool.lens_host), pool.max_pages * times + 2), -1, np.int32)
    table[:, :pool.max_pages] = pool.table_host[:, :pool.max_pages]
    used = -(-np.maximum(pool.lens_host, 0) // pool.page)
    table[np.arange(table.shape[1])[None] >= used[:, None]] = -1
    pool.table, pool.table_host, pool.max_pages = torch.from_numpy(table).cuda(), table, pool.max_pages * times
    c.batch = pool.batch(c.rows if tokens is None else tokens, getattr(c, "start", None))
    return c


def room(n):
    return torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("times", [4, 64])
@pytest.mark.parametrize("heads,kv_heads,hd,window", [(4, 1, 256, 0), (15, 5, 64, 0), (8, 2, 128, 60), (8, 1, 512, 0)])
@pytest.mark.parametrize("new,before,prefix", [([8] * 5, 40, 301), ([61, 33, 64, 40, 47], 70, 90), ([3, 1, 0, 5, 2] * 5, 33, 0)])
def test_trees_in_wide_tables(new, before, prefix, heads, kv_heads, hd, window, times):
    rng = np.random.default_rng(heads + hd + times)
    c = widen(TreeCall(rng, new, [before] * len(new), prefix, heads, kv_heads, hd, window=window), times)
    c.ws = room(c.kv.attention_tree_workspace(c.batch, heads))
    c.run().check()


@pytest.mark.parametrize("times", [4, 64])
@pytest.mark.parametrize("heads,kv_heads,hd,window", [(4, 1, 256, 0), (15, 5, 64, 0), (8, 2, 128, 60), (8, 1, 512, 0)])
@pytest.mark.parametrize("new,before", [([1] * 9, 90), ([700], 20), ([300, 1, 0, 280], 40)])
def test_weights_in_wide_tables(new, before, heads, kv_heads, hd, window, times):
    rng = np.random.default_rng(heads + hd + times)
    c = Weigh(rng, new, [before] * len(new), heads, kv_heads, hd, page=32, window=window)
    c.ldw = c.pool.max_pages * times * 32 + 3
    w = torch.rand(len(new), kv_heads, c.ldw)
    w[:, :, :c.w_host.shape[2]] = c.w_host
    c.w_host, c.w = w, w.cuda()
    widen(c, times)
    c.ws = room(c.kv.attention_weights_workspace(c.batch, heads))
    c.run().check()


@pytest.mark.parametrize("to", [False, True])
@pytest.mark.parametrize("times", [8, 64])
def test_evictions_in_wide_tables(times, to):
    """Tables of 2,560 and 20,480 rows, of which the sequences have up to 300."""
    rng = np.random.default_rng(times)
    c = Evict(rng, [300, 7, 0, 120, 250], 2, 64, 90, 20, to=to, separate=to)
    c.ldw = c.pool.max_pages * times * 16 + 5
    w = np.exp(2 * rng.standard_normal((5, 2, c.ldw))).astype(np.float32)
    c.w_host, c.w = w, torch.from_numpy(w.copy()).cuda()
    widen(c, times, tokens=5)
    c.test()


@pytest.mark.parametrize("new", [[1] * 5, [20, 3, 9, 1, 40]])
@pytest.mark.parametrize("times", [16, 300])
def test_blocks_in_wide_tables(times, new):
    """Some 200 blocks' and, past what registers hold, 3,000 blocks' room for a few."""
    rng = np.random.default_rng(times + len(new))
    c = BlockCall(rng, new, [130, 3, 0, 50, 100], 200, 4, 2, 128, 6).all_means()
    widen(c, times)
    c.ws = room(c.kv.attention_blocks_workspace(c.batch, 4, 6))
    c.run().check()


@pytest.mark.parametrize("heads,kv_heads,hd,dtype", [(32, 8, 128, "bf16"), (4, 1, 256, "f16"), (12, 12, 64, "f16"), (8, 1, 512, "bf16")])
def test_weights_of_a_prompt_among_single_tokens(heads, kv_heads, hd, dtype):
    """So few tokens a sequence that the prompt's rows pass a few at a time."""
    rng = np.random.default_rng(hd)
    Weigh(rng, [1] * 70 + [211] + [1] * 50, [50] * 70 + [90] + [70] * 50, heads, kv_heads, hd, dtype=dtype).run().check()
    Weigh(rng, [1] * 70 + [211] + [1] * 50, [50] * 70 + [90] + [70] * 50, heads, kv_heads, hd, dtype=dtype, window=77).run().check()


@pytest.mark.parametrize("prefix", [1000 * 16, 2042 * 16 + 5, 2043 * 16, 2043 * 16 + 1])
@pytest.mark.parametrize("give", [True, False])
def test_blocks_that_registers_hold_and_one_more(prefix, give):
    """1,005 blocks, 2,048 twice (a workgroup's eight values a thread), 2,049; many equal ones among them."""
    rng = np.random.default_rng(prefix)
    c = BlockCall(rng, [1, 1], [70, 9], prefix, 4, 2, 64, 40, give=give).all_means()
    c.run().check("as they come")
    c.means.copy_((c.means * 2).round() / 2)
    c.means[:, :, 1:] = 0
    c.run().check("many alike")


@pytest.mark.parametrize("nseq,kv_heads,hd", [(65, 8, 128), (33, 8, 512), (130, 8, 64)])
def test_lists_of_hundreds_of_blocks_chosen_ahead(nseq, kv_heads, hd):
    """More lists than the chip takes at once, with several values a thread."""
    rng = np.random.default_rng(nseq + hd)
    c = BlockCall(rng, [1] * nseq, rng.integers(0, 60, nseq), 700 * 16 + 3, kv_heads, kv_heads, hd, 3, dtype="bf16").all_means()
    c.run().check()
    c.means.copy_((c.means * 4).round())
    c.means[:, :, 2:] = 0
    c.run().check("many alike")


@pytest.mark.parametrize("to,separate", [(False, False), (True, True), (True, False)])
@pytest.mark.parametrize("n,keep,recent", [(9000, 17, 5), (9000, 4100, 300), (8193, 8192, 1)])
def test_rows_of_lists_past_the_registers_move(n, keep, recent, to, separate):
    """Tables of more than 8,192 rows: numbers, weights, K and V."""
    rng = np.random.default_rng(n + keep)
    Evict(rng, [n, n // 2, 3], 2, 64, keep, recent, page=256, to=to, separate=separate).test()
