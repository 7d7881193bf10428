"""omg_dev_attention_weights (PagedKv.attention_weights) against the plain
form in 64 bits, from given log sums: single tokens, prompts, ragged batches,
shared heads, windows, split queries, lengths short of the tokens, what
unseen rows hold, pages outside the pool, graphs.

Tolerance: a score is an f32 sum of exact products, off by at most 2^-20 of
sum |q k| scale (hd <= 512 terms in MFMA steps of 16 or 32); scale and the log
sum come in by one fma (half a step of its result, at most |score| + |lse| for
tiny ones: 2^-24), log2(e) by one product (2^-24 of the argument) and exp2 is off by
2^-22, so a probability by a factor 1 + d, d = 2^-19 size + 2^-23 (|lse| + size) +
2^-21; the f32 sum over r rows adds 2^-24 r (in steps: at most 2^-17 of the sum for
the rows here); the sum with the old weight rounds once, 2^-23 of both."""
from __future__ import annotations

import numpy as np
import pytest

import grande_amd as g
from paged import TYPES, Pool, starts
from test_shared_attention_gpu import SHAPES

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class Weigh:
    """One batch: `new` tokens a sequence after `before` own rows, with log sums of its own choice."""

    def __init__(self, rng, new, before, heads, kv_heads, hd, page=16, dtype="f16", window=0, tail=0, q_pad=0,
                 prefix=0, single=None):
        self.new = np.asarray(new)
        self.pool = Pool(rng, self.new + np.asarray(before), prefix, kv_heads, hd, page, dtype)
        self.heads, self.kv_heads, self.hd, self.window, self.dtype, self.page = heads, kv_heads, hd, window, dtype, page
        self.t, self.rows = int(self.new.sum()), int(self.new.sum()) + tail
        gen = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
        self.ldq = heads * hd + q_pad
        self.q = (1.7 * torch.randn(self.rows, self.ldq, generator=gen)).to(TYPES[dtype]).cuda()
        # log sums about as attention gives them: probabilities from tiny to over one
        self.lse = (3 + 2 * torch.randn(self.rows, heads, generator=gen)).cuda()
        self.scale = hd ** -0.5
        self.single = bool((self.new == 1).all()) and tail == 0 if single is None else single
        self.start = None if self.single else starts(self.new)
        self.batch, self.kv = self.pool.batch(self.rows, self.start), self.pool.kv()
        self.ldw = self.pool.max_pages * page + 3
        self.w_host = torch.randn(len(self.new), kv_heads, self.ldw, generator=gen).abs()
        self.w = self.w_host.cuda()
        self.ws = torch.full((self.kv.attention_weights_workspace(self.batch, heads),), 0xFF, dtype=torch.uint8, device="cuda")

    def run(self, stream=None):
        self.kv.attention_weights(self.batch, self.heads, self.q.data_ptr(), self.ldq, self.lse.data_ptr(), self.scale,
                                  self.w.data_ptr(), self.ldw, window=self.window,
                                  workspace=self.ws.data_ptr() if self.ws.numel() else None,
                                  workspace_bytes=self.ws.numel(), stream=stream)
        return self

    def expected(self, gone=lambda s, n: None):
        """(weights, tolerance, whether a row hears of a token) in 64 bits."""
        H, D, G, pool = self.heads, self.hd, self.heads // self.kv_heads, self.pool
        q, lse = self.q.double().cpu()[:, :H * D].view(self.rows, H, D), self.lse.double().cpu()
        w, tol = self.w_host.double().clone(), torch.zeros(self.w_host.shape, dtype=torch.float64)
        at = 0
        for s, n in enumerate(self.new.tolist()):
            length = int(pool.lens_host[s])
            k = pool.rows(pool.k_raw, s)
            own = length - n + torch.arange(n)
            key = torch.arange(length)
            see = key[None] <= own[:, None]
            if self.window:
                see &= own[:, None] - key[None] < self.window
            if gone(s, length) is not None:
                see &= ~gone(s, length)[None]
            for h in range(H):
                kh, l = k[:, h // G], lse[at:at + n, h]
                sc, size = q[at:at + n, h] @ kh.T * self.scale, q[at:at + n, h].abs() @ kh.abs().T * self.scale
                p = torch.where(see & (l > -np.inf)[:, None], (sc - l[:, None]).exp(), 0.0)
                d = 2.0 ** -19 * size + 2.0 ** -23 * (l.abs()[:, None] + size) + 2.0 ** -21 + 2.0 ** -17
                w[s, h // G, :length] += p.sum(0)
                tol[s, h // G, :length] += torch.where(p > 0, p * d, 0.0).sum(0)
            at += n
        return w, tol + 2.0 ** -23 * w

    def check(self, gone=lambda s, n: None, what=""):
        torch.cuda.synchronize()
        w, tol = self.expected(gone)
        got = self.w.double().cpu()
        for s in range(len(self.new)):
            n = max(0, int(self.pool.lens_host[s]))
            assert torch.equal(self.w[s, :, n:].cpu(), self.w_host[s, :, n:]), f"{what}: rows behind the last"
            off = (got[s, :, :n] - w[s, :, :n]).abs() - tol[s, :, :n]
            assert n == 0 or bool((off <= 0).all()), f"{what} sequence {s}: worst over its bound {float(off.max()):.3e}"
        return self


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES + [(40, 1, 64), (20, 1, 512)])
@pytest.mark.parametrize("nseq", [1, 9, 70])
def test_single_tokens(nseq, heads, kv_heads, hd, dtype):
    rng = np.random.default_rng(nseq * 100 + heads + hd)
    Weigh(rng, [1] * nseq, rng.integers(0, 90 if nseq > 1 else 900, nseq), heads, kv_heads, hd, dtype=dtype).run().check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES + [(40, 1, 64), (70, 2, 128)])
@pytest.mark.parametrize("new,before", [([40, 1, 0, 17, 64, 33], [0, 5, 7, 31, 2, 0]), ([300, 2], [0, 290]), ([2, 3, 0, 1, 5], [60, 0, 9, 100, 31])])
def test_ragged_batches(new, before, heads, kv_heads, hd, dtype):
    """Prompts, and a few tokens each: both kernels, keys that end inside a tile, diagonals."""
    rng = np.random.default_rng(heads + hd + len(new))
    Weigh(rng, new, before, heads, kv_heads, hd, page=32, dtype=dtype).run().check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("before", [0, 1, 15, 16, 255, 256, 257])
def test_lengths_and_pages(before, page):
    rng = np.random.default_rng(before + page)
    Weigh(rng, [1] * 3, [before, 0, 2 * before], 4, 2, 128, page=page).run().check()
    Weigh(rng, [70, 35], [before, 0], 4, 2, 64, page=page).run().check()


@pytest.mark.parametrize("window", [1, 7, 64, 300, (1 << 31) - 1])
@pytest.mark.parametrize("new,before", [([1] * 6, [0, 3, 60, 64, 100, 400]), ([130, 2, 50], [0, 90, 310]), ([3, 1, 0, 2] * 5, [9, 0, 4, 200] * 5)])
def test_windows(new, before, window):
    rng = np.random.default_rng(window % 1000 + len(new))
    Weigh(rng, new, before, 4, 1, 256, window=window).run().check()
    Weigh(rng, new, before, 6, 2, 64, window=window, dtype="bf16", page=32).run().check()


@pytest.mark.parametrize("heads,kv_heads,hd,rows", [(4, 1, 256, 1500), (2, 2, 128, 2000), (4, 2, 64, 1100), (2, 1, 512, 900)])
def test_long_prompts_with_split_queries(heads, kv_heads, hd, rows):
    rng = np.random.default_rng(hd)
    c = Weigh(rng, [rows], [100], heads, kv_heads, hd, page=64)
    assert c.ws.numel() > 0
    c.run().check()
    Weigh(rng, [rows, 0, rows // 3], [0, 50, 7], heads, kv_heads, hd, page=64, window=333).run().check()


def test_a_prefix_shifts_nothing():
    """Own rows alone are weighed, whatever prefix the sequences follow."""
    rng = np.random.default_rng(3)
    Weigh(rng, [1, 1, 1], [40, 0, 16], 4, 2, 64, prefix=100).run().check()
    Weigh(rng, [50, 40], [40, 0], 4, 2, 64, prefix=100, window=30).run().check()


def test_strides_and_rows_that_no_sequence_has():
    rng = np.random.default_rng(5)
    Weigh(rng, [3, 0, 1], [20, 4, 0], 4, 2, 128, tail=9, q_pad=24).run().check()
    Weigh(rng, [50, 45], [0, 4], 4, 4, 64, tail=70, q_pad=8).run().check()


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 35, 50, 33]])
def test_tokens_that_see_nothing_and_lengths_short_of_the_tokens(new):
    rng = np.random.default_rng(7)
    c = Weigh(rng, new, [20] * 4, 4, 2, 64)
    c.lse[1, 2] = -np.inf
    c.lse[c.t - 1] = -np.inf
    short = c.pool.lens_host.copy()
    short[1], short[2] = 0, (new[2] + 1) // 2
    c.pool.lens.copy_(torch.from_numpy(short))
    c.pool.lens_host = short
    c.run().check()
    c.w.copy_(c.w_host)
    c.pool.lens[1] = -(1 << 31)
    c.run().check()


@pytest.mark.parametrize("new", [[1] * 5, [33, 40, 36, 47, 50], [3, 1, 2, 4, 1]])
@pytest.mark.parametrize("hd", [64, 256, 512])
def test_what_other_rows_hold_does_not_matter(hd, new):
    """NaN and infinities in a key's row reach that row's weight alone; behind the last row none."""
    rng = np.random.default_rng(9)
    c = Weigh(rng, new, [10, 17, 30, 15, 40], 4, 2, hd, page=32, dtype="bf16")
    clean = c.run().w.clone()
    c.w.copy_(c.w_host)
    bad = {}
    for s in range(5):
        row = 3 + s
        bad[s] = row
        c.pool.k[int(c.pool.table_host[s, row // 32]), 0, row % 32] = float("nan") if s % 2 else float("inf")
        row = int(c.pool.lens_host[s])
        if row % 32:
            c.pool.k[int(c.pool.table_host[s, row // 32]), :, row % 32:] = float("nan")
    c.run()
    torch.cuda.synchronize()
    for s, row in bad.items():
        seen = row <= int(c.pool.lens_host[s]) - 1
        if seen and s % 2:
            assert bool(torch.isnan(c.w[s, 0, row]))
        c.w[s, 0, row] = clean[s, 0, row]
    assert torch.equal(c.w, clean)


def test_a_query_of_nan_reaches_the_rows_it_sees():
    rng = np.random.default_rng(11)
    for new in ([1, 1, 1], [40, 35, 50]):
        c = Weigh(rng, new, [20] * 3, 4, 2, 64)
        clean = c.run().w.clone()
        c.w.copy_(c.w_host)
        at = new[0] + new[1] // 2
        c.q[at, :64] = float("nan")  # head 0 of a token of sequence 1
        c.run()
        torch.cuda.synchronize()
        own = 20 + new[1] // 2
        assert bool(torch.isnan(c.w[1, 0, :own + 1]).all())
        c.w[1, 0, :own + 1] = clean[1, 0, :own + 1]
        assert torch.equal(c.w, clean)


def test_pages_outside_the_pool_keep_their_weights():
    rng = np.random.default_rng(13)
    for new in ([1] * 4, [35, 40, 50, 33], [3, 4, 1, 2]):
        c = Weigh(rng, new, [40, 60, 50, 45], 4, 2, 128, page=16)
        c.pool.table[0, 1], c.pool.table[1, 0], c.pool.table[1, 2] = c.pool.npages, -1, 1 << 30
        hidden = {0: [1], 1: [0, 2]}
        c.run().check(lambda s, n: torch.from_numpy(np.isin(np.arange(n) // 16, hidden.get(s, []))))


def test_lengths_past_the_table_stop_at_its_end():
    """The rows that the table reaches, with the tokens behind them."""
    rng = np.random.default_rng(15)
    c = Weigh(rng, [1, 1], [31, 31], 2, 1, 64, page=32)
    whole = c.run().w.clone()
    c.w.copy_(c.w_host)
    c.pool.lens[0] = 1000
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(whole, c.w)


@pytest.mark.parametrize("new", [[1] * 12, [700, 300], [40, 38, 50, 33, 61]])
def test_the_same_bits_each_time(new):
    """Eagerly, replayed behind other work on the same buffers, on another stream."""
    rng = np.random.default_rng(17)
    c = Weigh(rng, new, [50] * len(new), 4, 1, 256)
    first = c.run().w.clone()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        c.w.copy_(c.w_host)
        c.ws.random_(0, 256)
        if i == 2:
            side.wait_stream(torch.cuda.current_stream())
            c.run(side.cuda_stream)
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, c.w)


def test_pool_past_32_bit_offsets():
    rng = np.random.default_rng(19)
    npages, kv_heads, page, hd = 70_000, 2, 128, 256  # 9.2 GB of keys
    for new in ([1, 1], [70, 40]):
        c = Weigh(rng, new, [150, 129], 4, kv_heads, hd, page=page)
        near = c.run().w.clone()
        big = torch.zeros(npages, kv_heads, page, hd, dtype=torch.float16, device="cuda")
        place = rng.choice(np.arange(npages - 3000, npages), c.pool.npages, replace=False)
        big[torch.from_numpy(place).cuda()] = c.pool.k
        c.pool.table.copy_(torch.from_numpy(place.astype(np.int32)).cuda()[c.pool.table.long()])
        c.kv = g.PagedKv(big.data_ptr(), big.data_ptr(), npages, kv_heads, page, hd, g.ELEM_F16)
        c.w.copy_(c.w_host)
        c.run()
        torch.cuda.synchronize()
        assert torch.equal(near, c.w)
        del big


def test_more_lists_than_a_grids_second_dimension():
    """8,300 sequences of 33 tokens x 8 heads: each list's weights add up to its tokens."""
    nseq, n, heads, hd, page = 8300, 33, 8, 64, 16
    pages = -(-n // page)
    k, v = (torch.randn(nseq * pages, heads, page, hd, device="cuda").half() for _ in range(2))
    kv = g.PagedKv(k.data_ptr(), v.data_ptr(), nseq * pages, heads, page, hd, g.ELEM_F16)
    table = torch.arange(nseq * pages, dtype=torch.int32, device="cuda")
    lens = torch.full((nseq,), n, dtype=torch.int32, device="cuda")
    start = torch.arange(nseq + 1, dtype=torch.int32, device="cuda") * n
    b = g.PagedBatch(nseq, nseq * n, lens.data_ptr(), table.data_ptr(), pages, start.data_ptr())
    q = torch.randn(nseq * n, heads * hd, device="cuda").half()
    out, lse = torch.empty_like(q), torch.empty(nseq * n, heads, device="cuda")
    ws = torch.empty(max(16, kv.attention_workspace(b, heads)), dtype=torch.uint8, device="cuda")
    kv.attention(b, heads, q.data_ptr(), heads * hd, out.data_ptr(), heads * hd, hd ** -0.5, lse=lse.data_ptr(),
                 workspace=ws.data_ptr(), workspace_bytes=ws.numel())
    w = torch.zeros(nseq, heads, pages * page, device="cuda")
    assert kv.attention_weights_workspace(b, heads) == 0
    kv.attention_weights(b, heads, q.data_ptr(), heads * hd, lse.data_ptr(), hd ** -0.5, w.data_ptr(), pages * page)
    torch.cuda.synchronize()
    assert bool((w[:, :, n:] == 0).all())
    # (log sums off by 1e-6 + 2^-19 of scores' sums below 64, 33 additions)
    assert bool(((w.double().sum(-1) - n).abs() <= n * (2e-4 + 33 * 2.0 ** -22)).all())


def test_weights_of_attentions_own_log_sums_add_up_to_the_tokens():
    """Without a prefix each token gives its rows a weight of one in all, for each of its heads."""
    rng = np.random.default_rng(21)
    for new, window in (([1] * 9, 0), ([60, 33, 90], 0), ([60, 33, 90], 20)):
        c = Weigh(rng, new, [100] * len(new), 8, 2, 128, window=window)
        out = torch.empty_like(c.q)
        ws = torch.empty(c.kv.attention_workspace(c.batch, 8), dtype=torch.uint8, device="cuda")
        c.kv.attention(c.batch, 8, c.q.data_ptr(), c.ldq, out.data_ptr(), c.ldq, c.scale, window=window,
                       lse=c.lse.data_ptr(), workspace=ws.data_ptr() if ws.numel() else None, workspace_bytes=ws.numel())
        c.run()
        torch.cuda.synchronize()
        got = (c.w.double().cpu() - c.w_host.double()).sum(-1)
        exp = torch.from_numpy(np.repeat(np.asarray(new)[:, None] * 4.0, 2, 1))
        # lse is off by 1e-6 + 2^-19 size (|score| sums below 64 here), a weight's sum rounds 200 times
        assert bool(((got - exp).abs() <= exp * (2e-4 + 200 * 2.0 ** -22)).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(3, 1, 64), (8, 2, 128), (6, 2, 256), (7, 1, 512), (5, 5, 128), (40, 1, 64)])
@pytest.mark.parametrize("new,before,window", [([1, 1, 1], [700, 3, 290], 0), ([701], [0], 0), ([650, 3, 667], [9, 290, 40], 0),
                                               ([703, 690], [0, 33], 480)])
def test_keys_of_infinite_elements_that_score_minus_infinity_weigh_nothing(new, before, window, heads, kv_heads, hd, dtype):
    """exp(-inf) is 0, also from key blocks that whole tiles of tokens see, where
    heads leave rows of a tile over, a last tile has few tokens, and tokens that
    see nothing (a log sum of minus infinity) have queries of any kind."""
    rng = np.random.default_rng(heads + hd + len(new) + window)
    c = Weigh(rng, new, before, heads, kv_heads, hd, page=32, dtype=dtype, window=window)
    for s, n in enumerate(c.pool.lens_host.tolist()):
        for row in (0, 5, 40, 299, 300, n - 1):
            if row < n:
                c.pool.k[int(c.pool.table_host[s, row // 32]), row % kv_heads, row % 32, 7] = float("inf")
    c.q[:, 7::hd] = -c.q[:, 7::hd].abs() - 1
    idle = torch.from_numpy(rng.permutation(c.t)[:c.t // 5]).cuda()
    c.lse[idle] = -np.inf
    c.q[idle[0::3]] = float("nan")
    c.q[idle[1::3]] = float("inf")
    c.run().check()
