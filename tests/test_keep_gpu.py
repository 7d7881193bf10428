"""omg_dev_kv_keep (PagedKv.keep) and omg_dev_kv_evict (PagedKv.evict) against
numpy: moved rows bit for bit, everything else in the pool untouched; the
chosen rows and their weights exactly (they are copies)."""
from __future__ import annotations

import numpy as np
import pytest

import grande_amd as g
from paged import Pool

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


class Rows:
    """A pool of sequences, with `to` fresh pages a sequence for rows that move to other pages."""

    def __init__(self, rng, lens, kv_heads, hd, page=16, dtype="f16", to=0, page_pad=0):
        lens = np.asarray(lens)
        self.pool = Pool(rng, lens, 0, kv_heads, hd, page, dtype, spare=2 + to * len(lens), page_pad=page_pad)
        used = set(self.pool.table_host[s, i] for s in range(len(lens)) for i in range(-(-max(lens[s], 0) // page)))
        free = [p for p in range(self.pool.npages) if p not in used]
        self.to_host = np.asarray(free[:to * len(lens)], np.int32).reshape(len(lens), to) if to else None
        self.to = i32(self.to_host) if to else None
        self.kv, self.batch = self.pool.kv(), self.pool.batch(len(lens))
        self.n, self.kv_heads, self.page = len(lens), kv_heads, page

    def moved(self, raw, lists, first, table):
        """raw with row first[s] + j of head h being old row lists[s][h][j]."""
        old = raw.cpu()
        x, new = self.pool.view(old), old.clone()
        y = self.pool.view(new)
        for s in range(self.n):
            for h in range(self.kv_heads):
                rows = lists[s][h % len(lists[s])]
                for j, r in enumerate(rows):
                    if r < 0:
                        continue
                    d = int(first[s]) + j
                    a, b = int(self.pool.table_host[s, r // self.page]), int(table[s, d // self.page])
                    y[b, h, d % self.page] = x[a, h, r % self.page]
        return new

    def expect(self, lists, first=None, apart=False):
        first = np.zeros(self.n, int) if first is None else first
        table = self.to_host if apart else self.pool.table_host
        return [self.moved(x, lists, first, table) for x in (self.pool.k_raw, self.pool.v_raw)]

    def check(self, exp, what=""):
        torch.cuda.synchronize()
        for got, e in zip((self.pool.k_raw, self.pool.v_raw), exp):
            assert torch.equal(got.cpu().view(torch.int16), e.view(torch.int16)), what


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("nseq,kv_heads", [(1, 1), (5, 3), (130, 4)])
def test_paths_close_up_in_place(nseq, kv_heads, hd, dtype):
    """Accepted paths of drafts: rows of one list for all heads behind `first`, -1 behind the last."""
    rng = np.random.default_rng(nseq + hd)
    before, new = rng.integers(0, 40, nseq), rng.integers(1, 12, nseq)
    c = Rows(rng, before + new, kv_heads, hd, dtype=dtype)
    lists = np.full((nseq, 9), -1)
    for s in range(nseq):
        m = int(rng.integers(0, min(9, new[s]) + 1))
        lists[s, :m] = before[s] + np.sort(rng.permutation(new[s])[:m])
    exp = c.expect(lists[:, None], before)
    rows, first = i32(lists), i32(before)
    c.kv.keep(c.batch, rows.data_ptr(), 9, 9, first=first.data_ptr())
    c.check(exp)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 256), (512, 32)])
@pytest.mark.parametrize("nseq,kv_heads,count", [(3, 2, 1), (2, 1, 700), (40, 16, 90)])
def test_lists_of_each_head(nseq, kv_heads, count, hd, page, apart):
    """Random rows that ascend: few and many lists (slices of rows and whole ones in place), ends inside a page."""
    rng = np.random.default_rng(nseq + hd + count)
    lens = rng.integers(count, 2 * count + 40, nseq)
    c = Rows(rng, lens, kv_heads, hd, page=page, to=-(-count // page) if apart else 0, page_pad=24)
    lists = np.stack([np.stack([np.sort(rng.permutation(n)[:count]) for _ in range(kv_heads)]) for n in lens])
    lists[0, 0, count // 2:] = -1
    exp = c.expect(lists, apart=apart)
    padded = np.full((nseq * kv_heads, count + 3), 7)
    padded[:, :count] = lists.reshape(-1, count)
    rows = i32(padded)
    to = dict(to_table=c.to.data_ptr(), to_ld=c.to.shape[1]) if apart else {}
    c.kv.keep(c.batch, rows.data_ptr(), count + 3, count, per_head=True, **to)
    c.check(exp)
    if apart:  # what was read is as it was: the same again
        c.kv.keep(c.batch, rows.data_ptr(), count + 3, count, per_head=True, **to)
        c.check(exp)


def test_in_place_rows_run_over_their_own_lists():
    """Lists whose sources are others' places all the way: a shift by one, all rows, and every second one."""
    rng = np.random.default_rng(3)
    for nseq, kv_heads, hd in ((1, 1, 256), (300, 2, 64)):
        n = 1500 if nseq == 1 else 200
        c = Rows(rng, [n] * nseq, kv_heads, hd, page=32)
        for lists in (np.arange(1, n), np.arange(n), np.arange(0, n, 2)):
            exp = c.expect([[lists]] * nseq)
            rows = i32(np.tile(lists, (nseq, 1)))
            c.kv.keep(c.batch, rows.data_ptr(), len(lists), len(lists))
            c.check(exp, f"{len(lists)} rows")


@pytest.mark.parametrize("nseq,kv_heads,hd", [(1, 1, 256), (3, 2, 128), (300, 2, 64)])
def test_in_place_in_any_order(nseq, kv_heads, hd):
    """Lists that do not ascend, rows twice among them, none before its place."""
    rng = np.random.default_rng(4 + hd)
    n = 1200 if nseq < 10 else 150
    c = Rows(rng, [n] * nseq, kv_heads, hd, page=32)
    first = rng.integers(0, 20, nseq)
    count = n - 25
    lists = np.stack([[[int(rng.integers(first[s] + j, n)) for j in range(count)] for _ in range(kv_heads)] for s in range(nseq)])
    exp = c.expect(lists, first)
    rows, f = i32(lists.reshape(-1, count)), i32(first)
    c.kv.keep(c.batch, rows.data_ptr(), count, count, per_head=True, first=f.data_ptr())
    c.check(exp)


def test_to_other_pages_in_any_order_and_twice():
    rng = np.random.default_rng(5)
    c = Rows(rng, [50, 70], 2, 128, to=4)
    lists = np.stack([rng.integers(0, 50, 60), rng.integers(0, 70, 60)])
    exp = c.expect(lists[:, None], apart=True)
    rows = i32(lists)
    c.kv.keep(c.batch, rows.data_ptr(), 60, 60, to_table=c.to.data_ptr(), to_ld=4)
    c.check(exp)


def test_two_sequences_read_from_the_same_pages():
    """Forks: both read shared pages, each writes its own."""
    rng = np.random.default_rng(7)
    c = Rows(rng, [64, 64], 2, 64, to=2)
    c.pool.table[1] = c.pool.table[0]
    c.pool.table_host[1] = c.pool.table_host[0]
    lists = np.stack([np.sort(rng.permutation(64)[:30]), np.sort(rng.permutation(64)[:30])])
    exp = c.expect(lists[:, None], apart=True)
    rows = i32(lists)
    c.kv.keep(c.batch, rows.data_ptr(), 30, 30, to_table=c.to.data_ptr(), to_ld=2)
    c.check(exp)


@pytest.mark.parametrize("apart", [False, True])
def test_entries_that_move_nothing(apart):
    """Below zero, past the table, on pages outside the pool, to pages outside
    the pool, and in place ones that stand before their new place."""
    rng = np.random.default_rng(9)
    c = Rows(rng, [64, 64], 2, 64, to=2 if apart else 0)
    lists = np.tile(np.arange(4, 34), (2, 1))
    lists[0, 3], lists[0, 7], lists[1, 2], lists[1, 9] = -5, 1 << 30, 5 * 16, -1
    good = lists.copy()
    if not apart:
        lists[1, 20], good[1, 20] = 3, -1  # (row 20 keeps what it has)
    rows = lists.copy()
    # sequence 0's second page is outside the pool: rows 16 .. 31 neither go nor arrive
    old = c.pool.table_host.copy()
    c.pool.table[0, 1] = c.pool.npages
    if apart:
        c.to[1, 1] = -1
    good = np.where((good >= 5 * 16) | (good < 0), -1, good)
    for j in range(30):
        if 16 <= good[0, j] < 32 or (not apart and 16 <= j):
            good[0, j] = -1
        if apart and j >= 16:
            good[1, j] = -1
    exp = c.expect(good[:, None], apart=apart)
    r = i32(rows)
    to = dict(to_table=c.to.data_ptr(), to_ld=2) if apart else {}
    c.kv.keep(c.batch, r.data_ptr(), 30, 30, **to)
    c.check(exp)
    assert np.array_equal(old, c.pool.table_host)


def test_first_below_zero_and_past_the_table():
    rng = np.random.default_rng(11)
    c = Rows(rng, [40, 40, 40], 1, 64)
    lists = np.tile(np.arange(30, 40), (3, 1))
    good = lists.copy()
    good[0, :5] = -1  # places -5 .. -1
    good[1] = -1      # places past the table
    exp = c.expect(good[:, None], [-5, 0, 20])
    first = i32([-5, 1000, 20])
    c.kv.keep(c.batch, i32(lists).data_ptr(), 10, 10, first=first.data_ptr())
    c.check(exp)


# ------------------------------------------------------------------- evict

def choose(w, n, keep, recent):
    """The rows that stay of n with weights w, by their definition."""
    if n <= keep:
        return np.arange(n)
    old = n - recent
    key = np.where(np.isnan(w[:old]), -np.inf, w[:old].astype(np.float64))
    nan = np.isnan(w[:old])
    order = np.lexsort((np.arange(old), nan, -key))[:keep - recent]
    return np.concatenate([np.sort(order), np.arange(old, n)])


class Evict(Rows):
    def __init__(self, rng, lens, kv_heads, hd, keep, recent, weights=None, to=False, separate=False, **kw):
        page = kw.get("page", 16)
        super().__init__(rng, lens, kv_heads, hd, to=-(-keep // page) if to else 0, **kw)
        self.keep_n, self.recent, self.separate, self.lens = keep, recent, separate, np.asarray(lens)
        self.ldw = self.pool.max_pages * page + 5
        w = np.exp(2 * rng.standard_normal((self.n, kv_heads, self.ldw))).astype(np.float32)
        self.w_host = w if weights is None else weights(w)
        self.w = torch.from_numpy(self.w_host.copy()).cuda()
        self.kept = torch.full((self.n, kv_heads, keep + 9), 5.0, device="cuda") if separate else None
        self.rows = torch.full((self.n, kv_heads, keep), 77, dtype=torch.int32, device="cuda")

    def run(self, stream=None):
        kept = dict(kept_weights=self.kept.data_ptr(), kept_ld=self.keep_n + 9) if self.separate else {}
        to = dict(to_table=self.to.data_ptr(), to_ld=self.to.shape[1]) if self.to is not None else {}
        self.kv.evict(self.batch, self.keep_n, self.recent, self.w.data_ptr(), self.ldw, self.rows.data_ptr(), **kept,
                      **to, stream=stream)
        return self

    def expected(self):
        lists = [[choose(self.w_host[s, h], int(self.lens[s]), self.keep_n, self.recent) for h in range(self.kv_heads)]
                 for s in range(self.n)]
        w = self.w_host.copy()
        kept = np.full((self.n, self.kv_heads, self.keep_n + 9), 5.0, np.float32) if self.separate else w.copy()
        rows = np.full((self.n, self.kv_heads, self.keep_n), -1, np.int32)
        for s in range(self.n):
            for h in range(self.kv_heads):
                r, n = lists[s][h], int(self.lens[s])
                rows[s, h, :len(r)] = r
                kept[s, h, :len(r)] = w[s, h, r]
                if n > self.keep_n:
                    kept[s, h, self.keep_n:n] = 0.0
        return lists, rows, kept, w

    def check_all(self, exp, moved):
        lists, rows, kept, w = exp
        torch.cuda.synchronize()
        assert np.array_equal(self.rows.cpu().numpy(), rows)
        got = (self.kept if self.separate else self.w).cpu().numpy()
        assert np.array_equal(got.view(np.int32), kept.view(np.int32))
        if self.separate:
            assert np.array_equal(self.w.cpu().numpy().view(np.int32), w.view(np.int32))
        self.check(moved)

    def test(self):
        exp = self.expected()
        moved = self.expect(exp[0], apart=self.to is not None)
        self.run().check_all(exp, moved)


@pytest.mark.parametrize("to,separate", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (40, 8), (40, 0), (40, 40), (130, 64)])
@pytest.mark.parametrize("hd", [64, 256])
def test_the_heaviest_and_the_last_rows_stay(hd, keep, recent, to, separate):
    """Lengths of zero, up to keep, one past it and far past it; in place and on other pages."""
    rng = np.random.default_rng(keep + recent)
    Evict(rng, [0, 1, keep - 1, keep, keep + 1, keep + 100, 333, 1200], 2, hd, keep, recent, to=to, separate=separate).test()


def test_ties_go_to_the_first_rows():
    rng = np.random.default_rng(13)
    for make in (lambda w: np.zeros_like(w), lambda w: np.round(w), lambda w: np.where(w > 1, np.float32(2), -w * 0),
                 lambda w: np.floor(w * 2) % 3):
        for to in (False, True):
            Evict(rng, [300, 1000, 2000], 3, 64, 150, 20, weights=lambda w: make(w).astype(np.float32), to=to).test()


def test_weights_of_any_kind():
    """Infinities, NaN (chosen last), negatives, both zeros, denormals."""
    rng = np.random.default_rng(15)

    def make(w):
        kind = rng.integers(0, 8, w.shape)
        x = np.select([kind == i for i in range(7)], [w, -w, np.full_like(w, np.inf), np.full_like(w, -np.inf),
                                                      np.full_like(w, np.nan), np.zeros_like(w), -np.zeros_like(w)],
                      w * np.float32(1e-42))
        return x.astype(np.float32)
    for keep in (30, 500, 900):
        Evict(rng, [1000, 700], 2, 64, keep, 10, weights=make, to=True, separate=True).test()
        Evict(rng, [1000, 700], 2, 64, keep, 10, weights=make).test()


@pytest.mark.parametrize("n,keep", [(4096, 4095), (5000, 17), (65_536, 30_000), (65_537, 65_000), (150_001, 70_000)])
def test_long_lists(n, keep):
    """More rows than one part of the counting holds."""
    rng = np.random.default_rng(n)
    for to in (False, True):
        c = Evict(rng, [n], 1, 64, keep, min(keep, 100), page=256, to=to, separate=to)
        exp = c.expected()
        c.run()
        torch.cuda.synchronize()
        assert np.array_equal(c.rows.cpu().numpy(), exp[1])
        got = (c.kept if to else c.w).cpu().numpy()
        assert np.array_equal(got.view(np.int32), exp[2].view(np.int32))


@pytest.mark.parametrize("nseq,kv_heads", [(1, 1), (4, 8), (3, 11), (9, 4)])
@pytest.mark.parametrize("n,keep,recent,hd", [(300, 7, 2, 64), (4000, 1500, 900, 64), (6000, 3100, 1200, 128),
                                              (1000, 999, 0, 512)])
def test_choice_and_moves_in_one_launch_and_in_two(n, keep, recent, hd, nseq, kv_heads):
    """Lists that many workgroups choose from, each moving a slice of the rows, and more lists than that."""
    rng = np.random.default_rng(n + nseq)
    lens = rng.integers(keep // 2, n, nseq)
    lens[0] = n
    Evict(rng, lens, kv_heads, hd, keep, recent, page=64, to=True, separate=True).test()


def test_long_lists_of_equal_weights():
    rng = np.random.default_rng(17)
    c = Evict(rng, [140_000], 1, 64, 66_000, 5, page=256, weights=lambda w: np.ones_like(w))
    exp = c.expected()
    c.run()
    torch.cuda.synchronize()
    assert np.array_equal(c.rows.cpu().numpy(), exp[1]) and np.array_equal(c.w.cpu().numpy(), exp[2])


def test_lengths_past_the_table_and_below_zero():
    rng = np.random.default_rng(19)
    c = Evict(rng, [48, 48, 48], 2, 64, 20, 5, to=True, separate=True)
    c.lens = np.array([48, 0, 48])
    exp = c.expected()
    moved = c.expect(exp[0], apart=True)
    c.pool.lens.copy_(i32([5000, -3, 48]))
    c.run().check_all(exp, moved)


def test_evictions_captured_and_on_another_stream():
    """The same bits each time, also where a replay follows other work on the same buffers."""
    rng = np.random.default_rng(21)
    c = Evict(rng, rng.integers(100, 900, 9), 3, 128, 90, 30, to=True, separate=True)
    exp = c.expected()
    moved = c.expect(exp[0], apart=True)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    c.run().check_all(exp, moved)
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        c.rows.fill_(3)
        c.kept[:] = 5.0
        c.w.copy_(torch.from_numpy(c.w_host))
        if i == 2:
            side.wait_stream(torch.cuda.current_stream())
            c.run(side.cuda_stream)
        else:
            graph.replay()
        c.check_all(exp, moved)


def test_pool_past_32_bit_offsets():
    rng = np.random.default_rng(23)
    npages, kv_heads, page, hd = 40_000, 2, 128, 512  # 10.5 GB each for k and v
    raw = [torch.zeros(npages, kv_heads, page, hd, dtype=torch.float16, device="cuda") for _ in range(2)]
    table = rng.choice(np.arange(npages - 2000, npages), (2, 4), replace=False)
    to = rng.choice(np.arange(npages - 4000, npages - 2000), (2, 2), replace=False)
    for x in raw:
        x[torch.from_numpy(table.ravel()).cuda()] = torch.randn(8, kv_heads, page, hd, device="cuda").half()
    kv = g.PagedKv(raw[0].data_ptr(), raw[1].data_ptr(), npages, kv_heads, page, hd, g.ELEM_F16)
    lens, tab, to_d = i32([512, 400]), i32(table), i32(to)
    b = g.PagedBatch(2, 2, lens.data_ptr(), tab.data_ptr(), 4)
    lists = np.stack([np.sort(rng.permutation(400)[:200]) for _ in range(2)])
    r = i32(lists)
    want = [[x[torch.from_numpy(table[s, lists[s] // page]).cuda(), :, torch.from_numpy(lists[s] % page).cuda()].clone()
             for s in range(2)] for x in raw]
    kv.keep(b, r.data_ptr(), 200, 200, to_table=to_d.data_ptr(), to_ld=2)
    torch.cuda.synchronize()
    j = np.arange(200)
    for x, e in zip(raw, want):
        for s in range(2):
            assert torch.equal(x[torch.from_numpy(to[s, j // page]).cuda(), :, torch.from_numpy(j % page).cuda()], e[s])
    kv.keep(b, r.data_ptr(), 200, 200)
    torch.cuda.synchronize()
    for x, e in zip(raw, want):
        for s in range(2):
            assert torch.equal(x[torch.from_numpy(table[s, j // page]).cuda(), :, torch.from_numpy(j % page).cuda()], e[s])
