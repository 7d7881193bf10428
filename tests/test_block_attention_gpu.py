"""omg_dev_block_means and omg_dev_attention_blocks (PagedKv.block_means,
attention_blocks) against the plain form in 64 bits: pages that new rows touch,
scores and the blocks chosen (exactly: the same 64-bit sums, and ties to the
first ones), attention over their rows, prefixes that end inside a page,
several tokens a sequence, NaN and infinities, pages outside the pool, graphs.

Tolerance of the outputs: as for attention over a shared prefix, over the chosen
rows.  Means are f32 roundings of 64-bit sums: half a step.  Scores that lie
nearer to each other than 2^-20 of sum |q mean| may fall either way round (they
are compared as f32 here as there)."""
from __future__ import annotations

import numpy as np
import pytest

import grande_amd as g
from paged import TYPES, half_step
from test_shared_attention_gpu import SHAPES, Call, plain

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class BlockCall(Call):
    def __init__(self, rng, new, before, prefix, heads, kv_heads, hd, blocks, give=True, **kw):
        super().__init__(rng, new, before, prefix, heads, kv_heads, hd, **kw)
        self.blocks = blocks
        pool = self.pool
        self.means = torch.full((pool.npages, kv_heads, hd), 7.0, device="cuda")
        self.chosen = torch.full((self.rows, kv_heads, blocks), 77, dtype=torch.int32, device="cuda") if give else None
        self.ws = torch.full((self.kv.attention_blocks_workspace(self.batch, heads, blocks),), 0xFF, dtype=torch.uint8,
                             device="cuda")

    def all_means(self):
        """The means of the prefix's and the sequences' whole rows, by the calls that a program makes."""
        pool = self.pool
        if pool.prefix:
            n = torch.tensor([pool.prefix], dtype=torch.int32, device="cuda")
            start = torch.tensor([0, pool.prefix], dtype=torch.int32, device="cuda")
            b = g.PagedBatch(1, pool.prefix, n.data_ptr(), pool.prefix_table.data_ptr(), pool.prefix_table.numel(), start.data_ptr())
            self.kv.block_means(b, self.means.data_ptr())
        lens = np.maximum(pool.lens_host, 0)
        if lens.sum():
            start = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()
            self.kv.block_means(pool.batch(int(lens.sum()), start), self.means.data_ptr())
        torch.cuda.synchronize()
        return self

    def run(self, stream=None):
        self.kv.attention_blocks(self.batch, self.heads, self.q.data_ptr(), self.ldq, self.out.data_ptr(),
                                 self.heads * self.hd + 8, self.scale, self.means.data_ptr(), self.blocks,
                                 lse=self.lse.data_ptr(), chosen=self.chosen.data_ptr() if self.chosen is not None else None,
                                 workspace=self.ws.data_ptr(), workspace_bytes=self.ws.numel(), stream=stream)
        return self

    def choice(self, s, own, h, at, means):
        """The blocks that a token at row `own` of sequence s takes for KV head h."""
        page, P, G = self.pool.page, self.pool.prefix, self.heads // self.kv_heads
        np_ = -(-P // page)
        last = np_ + min(own, self.pool.max_pages * page - 1) // page
        ids = np.concatenate([self.pool.prefix_ids[:np_], self.pool.table.cpu().numpy()[s, :last - np_ + 1]]).astype(np.int64)
        bad = (ids < 0) | (ids >= self.pool.npages)
        q = self.q[at].double().cpu()[:self.heads * self.hd].view(self.kv_heads, G, self.hd)[h].sum(0)
        score = np.where(bad[:last], 0.0, (means[np.where(bad, 0, ids)[:last], h] @ q).numpy()).astype(np.float32)
        key = np.where(np.isnan(score), -np.inf, score)
        take = np.lexsort((np.arange(last), np.isnan(score), -key))[:self.blocks - 1]
        return np.append(np.sort(take), last), ids

    def check(self, what=""):
        torch.cuda.synchronize()
        hs = half_step(TYPES[self.dtype])
        pool, G, H, D, page, P = self.pool, self.heads // self.kv_heads, self.heads, self.hd, self.pool.page, self.pool.prefix
        np_ = -(-P // page)
        out = self.out[:, :H * D].double().cpu().view(self.rows, H, D)
        lse, q = self.lse.double().cpu(), self.q.double().cpu()[:, :H * D].view(self.rows, H, D)
        means, k, v = self.means.double().cpu(), pool.k.double().cpu(), pool.v.double().cpu()
        lens = pool.lens.cpu().numpy()
        at = 0
        for s, n in enumerate(self.new.tolist()):
            for i in range(n):
                own = int(lens[s]) - n + i
                if own < 0:
                    assert bool((out[at] == 0).all()) and bool((lse[at] == -np.inf).all())
                    if self.chosen is not None:
                        assert bool((self.chosen[at] == -1).all())
                    at += 1
                    continue
                for h in range(self.kv_heads):
                    take, ids = self.choice(s, own, h, at, means)
                    if self.chosen is not None:
                        got = self.chosen[at, h].cpu().numpy()
                        assert np.array_equal(got[:len(take)], take) and (got[len(take):] == -1).all(), f"{what} token {at} head {h}"
                    kk, vv = [], []
                    for b in take:
                        p = ids[b]
                        if not 0 <= p < pool.npages:
                            continue
                        end = min(page, P - b * page) if b < np_ else min(page, own + 1 - (b - np_) * page)
                        kk.append(k[p, h, :end])
                        vv.append(v[p, h, :end])
                    kk, vv = (torch.cat(x) if x else torch.zeros(0, D, dtype=torch.float64) for x in (kk, vv))
                    rows = slice(h * G, (h + 1) * G)
                    see = torch.ones(G, len(kk), dtype=torch.bool)
                    if not len(kk):
                        assert bool((out[at, rows] == 0).all()) and bool((lse[at, rows] == -np.inf).all())
                        continue
                    o, l, bound, size = plain(q[at, rows], kk, vv, see, self.scale)
                    tol = hs * (bound + o.abs()) + (2.0 ** -18 + 2.0 ** -19 * size[:, None]) * bound + 1e-7
                    off = (out[at, rows] - o).abs() - tol
                    assert bool((off <= 0).all()), f"{what} token {at} head {h}: worst over its bound {float(off.max()):.3e}"
                    assert bool(((lse[at, rows] - l).abs() <= 1e-6 + 2.0 ** -19 * size + 2.0 ** -21 * l.abs()).all())
                at += 1
        assert bool((self.out[:, H * D:] == 5.0).all()) and bool((self.out[at:] == 5.0).all())
        assert bool((self.lse[at:] == 5.0).all())
        if self.chosen is not None:
            assert bool((self.chosen[at:] == 77).all())
        return self


def mean_of(pool, table, n, page):
    """{page: mean [kv_heads][hd]} of a sequence of n rows, in 64 bits."""
    k = pool.k.double().cpu()
    return {int(table[j]): k[int(table[j]), :, :min(page, n - j * page)].mean(1) for j in range(-(-n // page))}


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_means_of_the_pages_that_new_rows_are_on(page, hd, dtype):
    rng = np.random.default_rng(page + hd)
    new, before = np.array([1, 3 * page + 1, 0, page, 5, 2]), np.array([0, 2 * page - 1, 7, page, page - 3, 4 * page])
    for single in (False, True):
        n = np.ones_like(new) if single else new
        c = BlockCall(rng, n, before + (new - n), 0, 4, 2, hd, 3, page=page, dtype=dtype, single=single)
        c.kv.block_means(c.batch, c.means.data_ptr())
        torch.cuda.synchronize()
        got, seen = c.means.double().cpu(), set()
        for s, m in enumerate(n.tolist()):
            length = int(c.pool.lens_host[s])
            for j, (p, mean) in enumerate(mean_of(c.pool, c.pool.table_host[s], length, page).items()):
                if m and j >= (length - m) // page:
                    seen.add(p)
                    assert bool(((got[p] - mean).abs() <= 2.0 ** -24 * mean.abs() + 2.0 ** -52).all()), (s, j)
        rest = [p for p in range(c.pool.npages) if p not in seen]
        assert bool((c.means[rest] == 7.0).all())


def test_means_of_lengths_short_of_the_tokens_and_pages_outside_the_pool():
    rng = np.random.default_rng(1)
    c = BlockCall(rng, [20, 3, 40], [0, 30, 10], 0, 4, 2, 64, 3)
    c.pool.lens.copy_(torch.tensor([7, 0, 50], dtype=torch.int32))
    c.pool.table[2, 1] = -1
    c.pool.table[2, 2] = c.pool.npages
    c.kv.block_means(c.batch, c.means.data_ptr())
    torch.cuda.synchronize()
    got = c.means.double().cpu()
    t = c.pool.table_host
    k = c.pool.k.double().cpu()
    exp = {int(t[0, 0]): k[int(t[0, 0]), :, :7].mean(1), int(t[2, 0]): k[int(t[2, 0])].mean(1), int(t[2, 3]): k[int(t[2, 3]), :, :2].mean(1)}
    for p in range(c.pool.npages):
        if p in exp:
            assert bool(((got[p] - exp[p]).abs() <= 2.0 ** -24 * exp[p].abs()).all())
        else:
            assert bool((got[p] == 7.0).all())


@pytest.mark.parametrize("evict", [False, True])
def test_means_and_blocks_of_rows_that_have_moved(evict):
    """An accepted path closed up over page borders, or an eviction: the means follow by a call whose new rows they are."""
    rng = np.random.default_rng(25)
    new, before, heads, kv_heads, hd = np.array([1, 40, 3, 37]), np.array([20, 30, 15, 64]), 4, 2, 64
    c = BlockCall(rng, new, before, 100, heads, kv_heads, hd, 3)
    c.all_means()
    pool = c.pool
    if evict:
        keep, max_len = 45, pool.max_pages * pool.page
        w = torch.rand(4 * kv_heads, max_len, device="cuda")
        rows = torch.empty(4, kv_heads, keep, dtype=torch.int32, device="cuda")
        c.kv.evict(c.batch, keep, 10, w.data_ptr(), max_len, rows.data_ptr())
        left = np.minimum(pool.lens_host, keep)
        moved = left
    else:
        rows = torch.full((4, 40), -1, dtype=torch.int32)
        took = [np.sort(rng.choice(n, -(-n // 2), replace=False)) for n in new]
        for s, x in enumerate(took):
            rows[s, :len(x)] = torch.from_numpy(before[s] + x)
        rows, first = rows.cuda(), torch.from_numpy(before.astype(np.int32)).cuda()
        c.kv.keep(c.batch, rows.data_ptr(), 40, 40, first=first.data_ptr())
        left = before + [len(x) for x in took]
        moved = new
    pool.lens.copy_(torch.from_numpy(left.astype(np.int32)))
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(moved)]).astype(np.int32)).cuda()
    c.kv.block_means(pool.batch(int(moved.sum()), start), c.means.data_ptr())
    torch.cuda.synchronize()
    got = c.means.double().cpu()
    for s in range(4):
        for p, mean in mean_of(pool, pool.table_host[s], int(left[s]), pool.page).items():
            assert bool(((got[p] - mean).abs() <= 2.0 ** -24 * mean.abs() + 2.0 ** -52).all()), (s, p)
    if evict:
        c.run().check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES + [(40, 1, 64), (36, 2, 128)])
@pytest.mark.parametrize("nseq,prefix,blocks", [(1, 1000, 9), (9, 301, 6), (5, 0, 3), (20, 77, 40)])
def test_single_tokens(nseq, prefix, blocks, heads, kv_heads, hd, dtype):
    """One token a sequence: prefixes that end inside a page, own rows from one up; fewer blocks than asked for."""
    rng = np.random.default_rng(nseq * 100 + heads + hd)
    BlockCall(rng, [1] * nseq, rng.integers(0, 90, nseq), prefix, heads, kv_heads, hd, blocks, dtype=dtype).all_means().run().check()


@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 1, 256), (6, 2, 64), (8, 1, 512)])
@pytest.mark.parametrize("new,before", [([3, 1, 0, 5, 2], [40, 0, 9, 31, 100]), ([40, 17, 33], [0, 70, 5])])
@pytest.mark.parametrize("prefix", [0, 200])
def test_several_tokens_a_sequence(prefix, new, before, heads, kv_heads, hd):
    """Every token its own list, none of a later block, and rows up to its own of the last."""
    rng = np.random.default_rng(heads + len(new) + prefix)
    BlockCall(rng, new, before, prefix, heads, kv_heads, hd, 4, dtype="bf16").all_means().run().check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("blocks", [1, 2, 5, 70])
def test_pages_and_numbers_of_blocks(blocks, page):
    rng = np.random.default_rng(page + blocks)
    BlockCall(rng, [1] * 3, [0, 3 * page, 5 * page + 1], 4 * page + 3, 4, 2, 128, blocks, page=page).all_means().run().check()


def test_many_blocks_and_long_lists():
    """More blocks than registers hold, lists split over work items, and the workspace's own list."""
    rng = np.random.default_rng(3)
    BlockCall(rng, [1, 1], [5, 40], 40_000, 2, 1, 64, 300).all_means().run().check()
    BlockCall(rng, [1], [20_000], 20_000, 2, 1, 64, 64).all_means().run().check()
    c = BlockCall(rng, [1, 1], [600, 40], 3000, 4, 2, 128, 20).all_means()
    c.run().check()
    first = c.out.clone(), c.lse.clone()
    c.chosen = None
    c.out[:, :-8], c.lse[:] = 0, 0
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(first[0], c.out) and torch.equal(first[1], c.lse)


@pytest.mark.parametrize("nseq,kv_heads,hd,blocks", [(64, 8, 128, 3), (57, 9, 128, 3), (32, 8, 512, 2), (43, 6, 512, 2),
                                                     (128, 8, 64, 3), (129, 8, 64, 3)])
def test_as_many_lists_as_the_chip_takes_at_once_and_more(nseq, kv_heads, hd, blocks):
    """Where the attention's workgroups choose for themselves, and one list more."""
    rng = np.random.default_rng(nseq + hd)
    BlockCall(rng, [1] * nseq, rng.integers(0, 60, nseq), 90, kv_heads, kv_heads, hd, blocks).all_means().run().check()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [[1] * 100, [20, 1, 3] * 33])
def test_many_scores(new, hd):
    """Launches of so many scores that a workgroup takes 64 blocks: the prefix's and sequences' of more than 64."""
    rng = np.random.default_rng(hd + len(new))
    before = rng.integers(0, 60, len(new))
    before[7] = 1200
    BlockCall(rng, new, before, 1100, 8, 8, hd, 4, dtype="bf16").all_means().run().check()


@pytest.mark.parametrize("give", [True, False])
@pytest.mark.parametrize("prefix", [251 * 16, 252 * 16 + 3, 2043 * 16 + 1, 2044 * 16 + 1])
def test_numbers_of_blocks_at_which_the_choice_changes(prefix, give):
    """A block a thread, several in registers, and more; equal scores among them; without the caller's list too."""
    rng = np.random.default_rng(prefix)
    c = BlockCall(rng, [1, 1], [70, 9], prefix, 4, 2, 64, 30, give=give).all_means()
    assert c.pool.max_pages == 5
    c.run().check("as they come")
    c.means.copy_((c.means * 2).round() / 2)
    c.means[:, :, 1:] = 0
    c.run().check("many alike")


def test_all_blocks_are_plain_attention():
    rng = np.random.default_rng(5)
    for new in ([1] * 5, [20, 3, 9]):
        c = BlockCall(rng, new, [40] * len(new), 100, 4, 2, 128, 30).all_means()
        c.run().check()
        mine, lse = c.out.clone(), c.lse.clone()
        c.ws = torch.empty(c.kv.attention_workspace(c.batch, 4), dtype=torch.uint8, device="cuda")
        Call.run(c)
        Call.check(c)
        # each rounds its probabilities and its result once (|v| < 6), and its sums
        assert bool(((mine - c.out).abs().float() <= 2.0 ** -10 * 6 + 2.0 ** -10 * c.out.abs().float()).all())
        assert bool(((lse - c.lse).abs() <= 1e-4).all())


def test_ties_go_to_the_first_blocks():
    rng = np.random.default_rng(7)
    c = BlockCall(rng, [1] * 3, [70, 20, 0], 200, 4, 2, 64, 6)
    c.all_means()
    c.means.zero_()
    c.run().check("all alike")
    c.means.copy_(torch.randint(-1, 2, c.means.shape[:1])[:, None, None].expand(c.means.shape).float())
    c.run().check("three kinds")


def test_scores_of_nan_and_infinity():
    """A NaN mean's block is chosen last; infinite ones first or last, by their sign."""
    rng = np.random.default_rng(9)
    c = BlockCall(rng, [1] * 4, [70, 20, 0, 33], 300, 2, 1, 64, 6).all_means()
    c.q.abs_()
    for i, x in enumerate((float("nan"), float("inf"), -float("inf"))):
        c.means[c.pool.prefix_table[2 + 4 * i:5 + 4 * i].long()] = x
    c.run().check()
    c.blocks = 6


def test_strides_and_rows_that_no_sequence_has():
    rng = np.random.default_rng(11)
    BlockCall(rng, [3, 0, 1], [20, 4, 0], 40, 4, 2, 128, 3, tail=9, q_pad=24).all_means().run().check()
    BlockCall(rng, [50, 45], [0, 4], 10, 4, 4, 64, 3, tail=70).all_means().run().check()


@pytest.mark.parametrize("new", [[1] * 4, [10, 5, 20, 3]])
def test_tokens_that_see_nothing(new):
    rng = np.random.default_rng(13)
    c = BlockCall(rng, new, [20] * 4, 0, 4, 2, 64, 3).all_means()
    short = c.pool.lens_host.copy()
    short[1], short[2] = 0, new[2] // 2
    c.pool.lens.copy_(torch.from_numpy(short))
    c.run().check()
    c.pool.lens[1] = -7
    c.run().check()


def test_pages_outside_the_pool_have_no_rows():
    rng = np.random.default_rng(15)
    for new in ([1] * 3, [20, 3, 9]):
        c = BlockCall(rng, new, [60, 70, 50], 50, 4, 2, 128, 4).all_means()
        c.pool.table[0, 1], c.pool.table[1, 0], c.pool.table[1, 2] = c.pool.npages, -1, 1 << 30
        c.run().check()


@pytest.mark.parametrize("new", [[1] * 4, [10, 5, 20, 3]])
@pytest.mark.parametrize("hd", [64, 256, 512])
def test_what_unseen_rows_hold_does_not_matter(hd, new):
    """NaN behind the last rows, in pages of nobody, and in blocks that are not chosen."""
    rng = np.random.default_rng(17)
    c = BlockCall(rng, new, [50, 37, 60, 45], 150, 4, 2, hd, 3, page=32, dtype="bf16", spare=4).all_means()
    c.run().check()
    want = c.out.clone(), c.lse.clone()
    taken = {(int(p), h) for h in range(2) for p in ()}
    ids = torch.cat([c.pool.prefix_table[None].expand(len(new), -1), c.pool.table], 1).cpu().numpy()
    at = 0
    for s, n in enumerate(new):
        for i in range(n):
            for h in range(2):
                taken |= {(int(ids[s, b]), h) for b in c.chosen[at, h].tolist() if b >= 0}
            at += 1
    for p in range(c.pool.npages):
        for h in range(2):
            if (p, h) not in taken:
                c.pool.k[p, h] = float("nan")
                c.pool.v[p, h] = float("inf")
    for s in range(4):
        n = int(c.pool.lens_host[s])
        if n % 32:
            p = int(c.pool.table_host[s, n // 32])
            c.pool.k[p, :, n % 32:], c.pool.v[p, :, n % 32:] = float("nan"), float("nan")
    p = int(c.pool.prefix_ids[150 // 32])
    c.pool.k[p, :, 150 % 32:], c.pool.v[p, :, 150 % 32:] = float("inf"), float("nan")
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(want[0], c.out) and torch.equal(want[1], c.lse)


def test_values_that_are_not_finite_and_sums_that_pass_f32():
    rng = np.random.default_rng(19)
    c = BlockCall(rng, [1] * 3, [40, 40, 40], 64, 4, 2, 128, 5, dtype="bf16").all_means()
    c.pool.v_raw.fill_(3.0e38)
    c.run()
    torch.cuda.synchronize()
    v = float(torch.tensor(3.0e38, dtype=torch.bfloat16).double())
    assert bool(((c.out[:, :512].double() - v).abs() <= 2 * half_step(torch.bfloat16) * v).all())
    c = BlockCall(rng, [1] * 3, [40, 40, 40], 64, 4, 2, 128, 5).all_means()
    own = int(c.pool.table_host[1, 2])
    sign = torch.where(torch.arange(128) % 2 == 0, 1.0, -1.0).half().cuda()
    c.pool.v[own, :, 3] = sign * float("inf")
    c.pool.k[int(c.pool.table_host[2, 2]), 0, 1] = float("nan")
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(c.out[1, :512], (sign * float("inf")).repeat(4))
    assert bool(torch.isnan(c.out[2, :256]).all()) and bool(torch.isfinite(c.out[2, 256:512]).all())
    assert bool(torch.isfinite(c.out[0, :512]).all())


@pytest.mark.parametrize("new", [[1] * 12, [9, 3]])
def test_the_same_bits_each_time(new):
    rng = np.random.default_rng(21)
    c = BlockCall(rng, new, [500] * len(new), 3000, 4, 1, 256, 20, page=64).all_means()
    c.run().check()
    first = c.out.clone(), c.lse.clone(), c.chosen.clone()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        c.kv.block_means(c.batch, c.means.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
        c.run(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        c.out[:, :-8], c.lse[:], c.chosen[:] = 0, 0, 3
        c.ws.random_(0, 256)
        if i == 2:
            side.wait_stream(torch.cuda.current_stream())
            c.run(side.cuda_stream)
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first[0], c.out) and torch.equal(first[1], c.lse) and torch.equal(first[2], c.chosen)


def test_pool_past_32_bit_offsets():
    rng = np.random.default_rng(23)
    npages, kv_heads, page, hd = 70_000, 2, 128, 256  # 9.2 GB each for k and v
    c = BlockCall(rng, [1, 1], [400, 300], 500, 4, kv_heads, hd, 4, page=page).all_means()
    near = c.run().out.clone()
    big = [torch.zeros(npages, kv_heads, page, hd, dtype=torch.float16, device="cuda") for _ in range(2)]
    place = rng.choice(np.arange(npages - 3000, npages), c.pool.npages, replace=False)
    for b, x in zip(big, (c.pool.k, c.pool.v)):
        b[torch.from_numpy(place).cuda()] = x
    d = torch.from_numpy(place.astype(np.int32)).cuda()
    c.pool.table.copy_(d[c.pool.table.long()])
    c.pool.prefix_table.copy_(d[c.pool.prefix_table.long()])
    c.kv = g.PagedKv(big[0].data_ptr(), big[1].data_ptr(), npages, kv_heads, page, hd, g.ELEM_F16)
    means = torch.zeros(npages, kv_heads, hd, device="cuda")
    means[torch.from_numpy(place).cuda()] = c.means
    c.means = means
    c.out.fill_(5.0)
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(near, c.out)
