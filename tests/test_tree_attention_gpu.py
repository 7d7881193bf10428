"""omg_dev_attention_tree (PagedKv.attention_tree) against the plain form in
64 bits: drafted trees and masks of any other kind, every tile shape, windows
by position, masks that leave nothing, masks shorter and longer than the
drafts, lengths short of the drafts, what unseen branches hold, graphs.

Tolerance: as for attention over a shared prefix (the same sums; a mask takes
keys out of them)."""
from __future__ import annotations

import numpy as np
import pytest

import grande_amd as g
from paged import TYPES, half_step
from test_shared_attention_gpu import SHAPES, Call, plain

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def tree_bits(rng, n):
    """Random parents: (sees [n][n], depth [n])."""
    see, depth = np.zeros((n, n), bool), np.zeros(n, np.int64)
    for i in range(n):
        parent = int(rng.integers(max(-1, i // 2 - 3), i))
        if parent >= 0:
            see[i], depth[i] = see[parent], depth[parent] + 1
        see[i, i] = True
    return see, depth


def random_bits(rng, n):
    """Any mask: half of all bits, later tokens' too, and some rows without one."""
    see = rng.random((n, n)) < 0.5
    see[rng.random(n) < 0.2] = False
    return see, rng.integers(0, n, n)


def packed(sees, words):
    """[t][words] int32 of each sequence's sees."""
    out = np.zeros((sum(len(x) for x in sees), words), np.uint32)
    at = 0
    for see in sees:
        for i, row in enumerate(see):
            for j in np.flatnonzero(row):
                if j // 32 < words:
                    out[at + i, j // 32] |= np.uint32(1 << (j % 32))
        at += len(see)
    return out.view(np.int32)


class TreeCall(Call):
    def __init__(self, rng, new, before, prefix, heads, kv_heads, hd, bits=tree_bits, words=None, junk=False, **kw):
        super().__init__(rng, new, before, prefix, heads, kv_heads, hd, **kw)
        made = [bits(rng, int(n)) for n in self.new]
        self.sees = [x for x, _ in made]
        self.words = words or max(1, (int(self.new.max()) + 31) // 32)
        m = packed(self.sees, self.words)
        if junk:  # bits behind each sequence's new tokens say nothing
            at = 0
            for see in self.sees:
                for i in range(len(see)):
                    for j in range(len(see), 32 * self.words):
                        m[at + i, j // 32] |= np.uint32(1 << (j % 32)).view(np.int32)
                at += len(see)
        m = np.concatenate([m, np.zeros((self.rows - self.t, self.words), np.int32)])
        self.mask = torch.from_numpy(m).cuda()
        # positions of a tree: depth behind the rows before
        self.pos_host = [self.pool.prefix + int(self.pool.lens_host[s]) - int(n) + d
                         for s, (n, (_, d)) in enumerate(zip(self.new, made))]
        p = np.concatenate(self.pos_host + [np.zeros(self.rows - self.t, np.int64)])
        self.positions = torch.from_numpy(p.astype(np.int32)).cuda()
        self.ws = torch.full((self.kv.attention_tree_workspace(self.batch, heads),), 0xFF, dtype=torch.uint8, device="cuda")

    def run(self, stream=None):
        self.kv.attention_tree(self.batch, self.heads, self.q.data_ptr(), self.ldq, self.out.data_ptr(),
                               self.heads * self.hd + 8, self.scale, self.mask.data_ptr(), self.words,
                               window=self.window, positions=self.positions.data_ptr() if self.window else None,
                               lse=self.lse.data_ptr(), workspace=self.ws.data_ptr() if self.ws.numel() else None,
                               workspace_bytes=self.ws.numel(), stream=stream)
        return self

    def see(self, s):
        """[n][prefix + length]: the keys that each new token of sequence s sees."""
        n, P, length = int(self.new[s]), self.pool.prefix, int(self.lens_now[s])
        key, base = np.arange(P + length), length - n
        see = np.zeros((n, P + length), bool)
        old = key < P + max(base, 0)
        see[:, old] = True
        if self.window:
            see[:, old] &= self.pos_host[s][:, None] - key[None, old] < self.window
        for j in range(max(0, -base), min(n, 32 * self.words)):
            see[:, P + base + j] = self.sees[s][:, j]
        return torch.from_numpy(see)

    def check(self, what="", skip_keys=lambda seq, own: None):
        torch.cuda.synchronize()
        hs = half_step(TYPES[self.dtype])
        pool, G, H, D = self.pool, self.heads // self.kv_heads, self.heads, self.hd
        self.lens_now = pool.lens.cpu().numpy()
        pool.lens_host = self.lens_now
        out = self.out[:, :H * D].double().cpu().view(self.rows, H, D)
        lse, q = self.lse.double().cpu(), self.q.double().cpu()[:, :H * D].view(self.rows, H, D)
        pk, pv = pool.prefix_rows(pool.k_raw), pool.prefix_rows(pool.v_raw)
        at = 0
        for s, n in enumerate(self.new):
            n = int(n)
            ok, ov = (torch.cat([a, pool.rows(x, s)]) for a, x in ((pk, pool.k_raw), (pv, pool.v_raw)))
            see = self.see(s)
            gone = skip_keys(s, int(self.lens_now[s]))
            if gone is not None:
                see[:, pool.prefix:] &= ~gone[None]
            for h in range(H):
                k, v = ok[:, h // G], ov[:, h // G]
                nan = ~(torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1))  # (rows of NaN that nobody sees)
                assert not bool((see & nan[None]).any()) or what == "NaN"
                k, v = torch.where(nan[:, None], 0.0, k), torch.where(nan[:, None], 0.0, v)
                o, l, bound, size = plain(q[at:at + n, h], k, v, see, self.scale)
                got, got_l = out[at:at + n, h], lse[at:at + n, h]
                spoilt = (see & nan[None]).any(1)
                assert bool(torch.isnan(got[spoilt]).all())
                tol = hs * (bound + o.abs()) + (2.0 ** -18 + 2.0 ** -19 * size[:, None]) * bound + 1e-7
                off = ((got - o).abs() - tol)[~spoilt]
                assert bool((off <= 0).all()), f"{what} sequence {s} head {h}: worst over its bound {float(off.max()):.3e}"
                empty = torch.isinf(l) & ~spoilt
                full = ~torch.isinf(l) & ~spoilt
                assert bool((got_l[empty] == -np.inf).all()) and bool((got[empty] == 0).all())
                assert bool(((got_l - l).abs()[full] <= 1e-6 + 2.0 ** -19 * size[full] + 2.0 ** -21 * l[full].abs()).all()), f"{what} lse"
            at += n
        assert bool((self.out[:, H * D:] == 5.0).all()) and bool((self.out[at:] == 5.0).all())
        assert bool((self.lse[at:] == 5.0).all())
        return self


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
@pytest.mark.parametrize("new,before,prefix", [([8] * 5, 40, 301), ([3, 1, 0, 5, 2] * 5, 33, 65), ([61, 33, 64, 40, 47], 70, 90)])
def test_trees(new, before, prefix, heads, kv_heads, hd, dtype):
    """Own items (few rows a sequence) and tiles that hold whole drafts; bases that end inside a tile."""
    rng = np.random.default_rng(heads + hd + len(new))
    TreeCall(rng, new, before + rng.integers(0, 20, len(new)), prefix, heads, kv_heads, hd, dtype=dtype).run().check()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("new,before", [([5, 9, 1, 4], [0, 1, 31, 32]), ([70, 33, 65], [0, 17, 64]), ([2] * 9, [0] * 9)])
@pytest.mark.parametrize("prefix", [0, 50])
def test_any_mask(prefix, new, before, hd):
    """Half of all bits: later tokens seen, tokens that do not see themselves,
    rows that see nothing (with neither prefix nor rows before: zeros and -infinity)."""
    rng = np.random.default_rng(hd + sum(new))
    TreeCall(rng, new, before, prefix, 4, 2, hd, page=32, bits=random_bits).run().check()


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_masks_shorter_and_longer_than_the_drafts(hd):
    rng = np.random.default_rng(3 + hd)
    for new in ([70, 40, 5], [3, 40, 1, 2]):
        TreeCall(rng, new, [20] * len(new), 30, 4, 2, hd, words=1).run().check()
        TreeCall(rng, new, [20] * len(new), 30, 4, 2, hd, words=5, junk=True).run().check()


@pytest.mark.parametrize("window", [1, 7, 64, 300])
@pytest.mark.parametrize("new,before", [([8] * 6, [0, 3, 60, 64, 100, 400]), ([50, 33, 64], [0, 90, 310])])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 1, 256), (6, 2, 64), (8, 1, 512)])
def test_windows_count_back_from_the_positions(heads, kv_heads, hd, new, before, window):
    rng = np.random.default_rng(window + len(new))
    TreeCall(rng, new, before, 200, heads, kv_heads, hd, window=window, dtype="bf16", page=32).run().check()
    TreeCall(rng, new, before, 0, heads, kv_heads, hd, window=window, bits=random_bits).run().check()


@pytest.mark.parametrize("window", [1, 100, 700, 10_000])
@pytest.mark.parametrize("heads,kv_heads,hd,new,before", [(4, 1, 256, [3, 9, 1], [40, 0, 130]), (8, 2, 64, [61, 40, 20], [5, 300, 0]),
                                                          (8, 1, 512, [5, 7], [20, 9]), (16, 2, 128, [33] * 30, [3] * 30)])
def test_windows_at_the_end_of_long_prefixes(heads, kv_heads, hd, new, before, window):
    """The splits share out what a tile sees, from near its end to all of it; sums that f32 does not hold too."""
    rng = np.random.default_rng(window + hd)
    c = TreeCall(rng, new, before, 5003, heads, kv_heads, hd, window=window, dtype="bf16", page=64)
    c.run().check()
    for s in range(0, len(new), 2):  # (positions that lie far back see more)
        c.pos_host[s] = c.pos_host[s] - rng.integers(0, 6000, len(c.pos_host[s]))
    c.positions.copy_(torch.from_numpy(np.concatenate(c.pos_host).astype(np.int32)))
    c.run().check("far back")
    c.pool.v_raw.fill_(3.0e38)
    c.run()
    torch.cuda.synchronize()
    v = float(torch.tensor(3.0e38, dtype=torch.bfloat16).double())
    assert bool(((c.out[:, :heads * hd].double() - v).abs() <= 2 * half_step(torch.bfloat16) * v).all())


def test_single_tokens_without_start():
    rng = np.random.default_rng(5)
    c = TreeCall(rng, [1] * 7, rng.integers(0, 50, 7), 20, 4, 2, 128, bits=random_bits)
    assert c.single
    c.run().check()


@pytest.mark.parametrize("new", [[40, 35, 50, 33], [8, 5, 3, 6]])
def test_lengths_short_of_the_drafts(new):
    """Rows that a draft has no room for are seen by nobody; a length of zero, and below, has none."""
    rng = np.random.default_rng(7)
    for prefix in (0, 33):
        c = TreeCall(rng, new, [20] * 4, prefix, 4, 2, 64, bits=random_bits)
        short = c.pool.lens_host.copy()
        short[1], short[2] = 0, new[2] // 2
        c.pool.lens.copy_(torch.from_numpy(short))
        c.run().check()
        c.pool.lens[1] = -(1 << 31)
        c.out[:, :-8] = 0
        c.run()
        torch.cuda.synchronize()
        at = new[0]
        c.pool.lens[1] = 0
        kept = c.out[at:at + new[1]].clone()
        c.run()
        torch.cuda.synchronize()
        assert torch.equal(kept, c.out[at:at + new[1]])


def test_strides_and_rows_that_no_sequence_has():
    rng = np.random.default_rng(9)
    TreeCall(rng, [3, 0, 6], [20, 4, 0], 40, 4, 2, 128, tail=9, q_pad=24).run().check()
    TreeCall(rng, [50, 45], [0, 4], 10, 4, 4, 64, tail=70).run().check()


@pytest.mark.parametrize("new", [[40, 35, 50, 33], [8, 5, 3, 6]])
@pytest.mark.parametrize("hd", [64, 256, 512])
def test_other_branches_of_nan_do_not_matter(hd, new):
    """A new row of NaN reaches the tokens whose bits have it and no others."""
    rng = np.random.default_rng(11)
    c = TreeCall(rng, new, [17, 30, 15, 40], 77, 4, 2, hd, page=32, dtype="bf16")
    for s in range(4):
        row = int(c.pool.lens_host[s]) - new[s] + new[s] // 2
        at = int(c.pool.table_host[s, row // 32])
        c.pool.k[at, :, row % 32] = float("nan")
        c.pool.v[at, :, row % 32] = float("nan")
        row = int(c.pool.lens_host[s])  # behind the last row
        if row % 32:
            c.pool.v[int(c.pool.table_host[s, row // 32]), :, row % 32:] = float("inf")
    c.run().check("NaN")


def test_pages_outside_the_pool_are_not_seen():
    rng = np.random.default_rng(13)
    for new in ([35, 40, 50, 33], [3, 4, 1, 2]):
        c = TreeCall(rng, new, [40, 60, 50, 45], 50, 4, 2, 128, page=16)
        c.pool.table[0, 1], c.pool.table[1, 0], c.pool.table[1, 2] = c.pool.npages, -1, 1 << 30
        hidden = {0: [1], 1: [0, 2]}
        c.run().check(skip_keys=lambda s, n: torch.from_numpy(np.isin(np.arange(n) // 16, hidden.get(s, []))))


def test_means_of_values_whose_sums_pass_f32():
    """bf16 values near the type's largest: a mean of finite values is finite."""
    rng = np.random.default_rng(15)
    for new in ([8] * 4, [40] * 4):
        c = TreeCall(rng, new, [60] * 4, 40, 4, 2, 128, dtype="bf16")
        c.pool.v_raw.fill_(3.0e38)
        c.run()
        torch.cuda.synchronize()
        got = c.out[:, :512].double()
        v = float(torch.tensor(3.0e38, dtype=torch.bfloat16).double())
        assert bool(((got - v).abs() <= 2 * half_step(torch.bfloat16) * v).all())


@pytest.mark.parametrize("new", [[8] * 12, [61, 40, 33], [3, 2, 5, 1] * 3])
def test_long_bases_split_captured_and_repeated(new):
    """Splits and their join, the same bits each time, eagerly, replayed and on another stream."""
    rng = np.random.default_rng(17 + len(new))
    c = TreeCall(rng, new, [700] * len(new), 900, 4, 1, 256, page=64)
    c.run().check()
    first = c.out.clone(), c.lse.clone()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        c.out[:, :-8], c.ws[:] = 0, 0x7F
        c.lse.zero_()
        if i == 3:
            side.wait_stream(torch.cuda.current_stream())
            c.run(side.cuda_stream)
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first[0], c.out) and torch.equal(first[1], c.lse)


def test_a_causal_mask_is_plain_attention():
    """Bits up to the token's own: what `attention` gives, within the two calls' roundings."""
    rng = np.random.default_rng(19)
    causal = lambda rng, n: (np.tril(np.ones((n, n), bool)), np.arange(n))
    for new, window in (([9, 3, 17], 0), ([9, 3, 17], 30), ([50, 40, 33], 0), ([50, 40, 33], 64)):
        c = TreeCall(rng, new, [40, 100, 7], 60, 4, 2, 128, bits=causal, window=window, dtype="bf16")
        causal_in_window = window >= max(new) or not window
        tree = c.run().out.clone()
        if causal_in_window:
            Call.check(Call.run(c), "plain")
            # each rounds its probabilities and its result once: two steps of sum p |v| (|v| < 6)
            assert bool(((tree - c.out).abs().float() <= 2.0 ** -7 * 6).all())
