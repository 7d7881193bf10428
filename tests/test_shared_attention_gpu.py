"""omg_dev_attention_shared (PagedKv.attention) against the plain form in 64
bits: every tile shape (few and many query rows, single tokens and prompts),
pages, windows, ragged batches, rows that see nothing, lengths of zero, what
unseen cache rows hold, pools past 32-bit offsets, graphs and streams.

Tolerance: the probabilities are rounded to the cache's type (half a step of
each, so at most half a step of sum p |v|), the output once more; scores are
f32 sums whose error, below 2^-20 of sum |q k| scale, enters p as a factor;
the f32 sums over keys stay below 2^-18 of sum p |v|."""
from __future__ import annotations

import numpy as np
import pytest

import grande_amd as g
from paged import TYPES, Pool, half_step, starts

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def plain(q, k, v, see, scale):
    """[rows][hd] queries over [keys][hd] in 64 bits: out, lse, the bound sum p |v|, and the scores' size."""
    s = (q @ k.T) * scale
    size = ((q.abs() @ k.abs().T) * scale).masked_fill(~see, 0.0).amax(-1) if k.shape[0] else torch.zeros(len(q))
    s = s.masked_fill(~see, -np.inf)
    v = torch.where(see.any(0)[:, None], v, torch.zeros_like(v))
    m = s.amax(-1, keepdim=True) if k.shape[0] else torch.full((len(q), 1), -np.inf)
    p = (s - torch.where(torch.isinf(m), torch.zeros_like(m), m)).exp()
    l = p.sum(-1, keepdim=True)
    safe = torch.where(l > 0, l, torch.ones_like(l))
    out, bound = (p / safe) @ v, (p / safe) @ v.abs()
    lse = torch.where(l[:, 0] > 0, m[:, 0] + safe[:, 0].log(), torch.full_like(l[:, 0], -np.inf))
    return out, lse, bound, size


class Call:
    """One batch on the GPU: `new` tokens a sequence after `before` own rows."""

    def __init__(self, rng, new, before, prefix, heads, kv_heads, hd, page=16, dtype="f16", window=0, tail=0,
                 single=None, q_pad=0, spare=2, qscale=1.7):
        self.new, self.before = np.asarray(new), np.asarray(before)
        self.pool = Pool(rng, self.new + self.before, prefix, kv_heads, hd, page, dtype, spare=spare)
        self.heads, self.kv_heads, self.hd, self.window, self.dtype = heads, kv_heads, hd, window, dtype
        self.t = int(self.new.sum())
        self.rows = self.t + tail
        gen = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
        self.ldq = heads * hd + q_pad
        self.q = (qscale * torch.randn(self.rows, self.ldq, generator=gen)).to(TYPES[dtype]).cuda()
        self.out = torch.full((self.rows, heads * hd + 8), 5.0, dtype=TYPES[dtype], device="cuda")
        self.lse = torch.full((self.rows, heads), 5.0, device="cuda")
        self.scale = hd ** -0.5
        self.single = bool((self.new == 1).all()) and tail == 0 if single is None else single
        self.start = None if self.single else starts(self.new)
        self.batch = self.pool.batch(self.rows, self.start)
        self.kv = self.pool.kv()
        self.ws = torch.full((self.kv.attention_workspace(self.batch, heads),), 0xFF, dtype=torch.uint8, device="cuda")

    def run(self, stream=None):
        self.kv.attention(self.batch, self.heads, self.q.data_ptr(), self.ldq, self.out.data_ptr(),
                          self.heads * self.hd + 8, self.scale, window=self.window, lse=self.lse.data_ptr(),
                          workspace=self.ws.data_ptr() if self.ws.numel() else None, workspace_bytes=self.ws.numel(),
                          stream=stream)
        return self

    def check(self, what="", skip_keys=lambda seq, own: None):
        """skip_keys(seq, n): own rows of a sequence that the call leaves out (a bool mask), if any."""
        torch.cuda.synchronize()
        hs = half_step(TYPES[self.dtype])
        pool, G, H, D = self.pool, self.heads // self.kv_heads, self.heads, self.hd
        out = self.out[:, :H * D].double().cpu().view(self.rows, H, D)
        lse, q = self.lse.double().cpu(), self.q.double().cpu()[:, :H * D].view(self.rows, H, D)
        pk, pv = pool.prefix_rows(pool.k_raw), pool.prefix_rows(pool.v_raw)
        P, at = pool.prefix, 0
        for s, n in enumerate(self.new):
            length = int(pool.lens_host[s])
            ok, ov = (torch.cat([a, pool.rows(x, s)]) for a, x in ((pk, pool.k_raw), (pv, pool.v_raw)))
            pos = P + length - n + torch.arange(int(n))
            key = torch.arange(P + length)
            see = key[None] <= pos[:, None]
            if self.window:
                see &= pos[:, None] - key[None] < self.window
            gone = skip_keys(s, length)
            if gone is not None:
                see[:, P:] &= ~gone[None]
            for h in range(H):
                o, l, bound, size = plain(q[at:at + n, h], ok[:, h // G], ov[:, h // G], see, self.scale)
                got, got_l = out[at:at + n, h], lse[at:at + n, h]
                tol = hs * (bound + o.abs()) + (2.0 ** -18 + 2.0 ** -19 * size[:, None]) * bound + 1e-7
                off = (got - o).abs() - tol
                assert bool((off <= 0).all()), \
                    f"{what} sequence {s} head {h}: off by {float((got - o).abs().max()):.3e}, worst over its bound {float(off.max()):.3e}"
                empty = torch.isinf(l)
                assert torch.equal(torch.isinf(got_l), empty) and bool((got_l[empty] < 0).all())
                assert bool(((got_l - l).abs()[~empty] <= 1e-6 + 2.0 ** -19 * size[~empty] + 2.0 ** -21 * l[~empty].abs()).all()), f"{what} lse"
            at += int(n)
        assert bool((self.out[:, H * D:] == 5.0).all()) and bool((self.out[at:] == 5.0).all())
        assert bool((self.lse[at:] == 5.0).all())
        return self


SHAPES = [(4, 1, 256), (4, 2, 128), (8, 1, 512), (3, 3, 64), (15, 5, 64), (14, 2, 128), (2, 1, 256)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
@pytest.mark.parametrize("nseq", [1, 9, 70])
def test_single_tokens(nseq, heads, kv_heads, hd, dtype):
    """A decoding step: 1 to 70 sequences over a prefix that ends inside a page, own rows from one up."""
    rng = np.random.default_rng(nseq * 100 + heads + hd)
    Call(rng, [1] * nseq, rng.integers(0, 90, nseq), 301, heads, kv_heads, hd, dtype=dtype).run().check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
def test_ragged_questions(heads, kv_heads, hd, dtype):
    rng = np.random.default_rng(heads + hd)
    Call(rng, [40, 1, 0, 17, 64, 33], [0, 5, 7, 31, 2, 0], 200, heads, kv_heads, hd, page=32, dtype=dtype).run().check()


@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
def test_a_few_tokens_each(heads, kv_heads, hd):
    """Two to five tokens a sequence: own rows in work items of their own, found through start."""
    rng = np.random.default_rng(heads * 3 + hd)
    new = rng.integers(0, 6, 21)
    Call(rng, new, rng.integers(0, 70, 21), 65, heads, kv_heads, hd, page=64).run().check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 33, 1000])
def test_prefix_lengths_and_pages(prefix, page):
    rng = np.random.default_rng(prefix + page)
    Call(rng, [1] * 5, [0, 1, 15, 16, 300], prefix, 4, 2, 128, page=page, dtype="bf16").run().check()


@pytest.mark.parametrize("window", [1, 7, 64, 300])
@pytest.mark.parametrize("new,before", [([1] * 6, [0, 3, 60, 64, 100, 400]), ([30, 2, 50], [0, 90, 10]),
                                        ([3, 1, 0, 2] * 5, [9, 0, 4, 200] * 5)])
def test_windows(new, before, window):
    rng = np.random.default_rng(window + len(new))
    Call(rng, new, before, 200, 4, 1, 256, window=window).run().check()
    Call(rng, new, before, 333, 6, 2, 64, window=window, dtype="bf16", page=32).run().check()


@pytest.mark.parametrize("heads,kv_heads,hd,rows", [(4, 1, 256, 700), (2, 2, 128, 900), (4, 2, 64, 1100), (1, 1, 512, 300)])
def test_long_prompts_without_a_prefix(heads, kv_heads, hd, rows):
    rng = np.random.default_rng(hd)
    Call(rng, [rows, 65], [0, 10], 0, heads, kv_heads, hd, page=64).run().check()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_many_tiles_run_through_prefix_and_own_keys(hd):
    """Enough rows that a tile takes the prefix and its sequences' own keys in one item."""
    rng = np.random.default_rng(hd + 1)
    n = 40 if hd == 512 else 70
    Call(rng, rng.integers(30, 60, n), rng.integers(0, 20, n), 90, 16, 8, hd, page=32, dtype="bf16").run().check()


def test_many_query_heads_on_one_key_head():
    rng = np.random.default_rng(21)
    Call(rng, [1] * 3, [10, 33, 0], 70, 40, 1, 64).run().check()
    Call(rng, [2, 1, 0, 3], [10, 33, 0, 4], 0, 40, 1, 128).run().check()


def test_long_own_rows_are_split_and_joined():
    rng = np.random.default_rng(23)
    Call(rng, [1, 1, 1], [5000, 0, 2500], 0, 4, 2, 128, page=128).run().check()
    Call(rng, [9], [4000], 3000, 2, 1, 256, page=64, dtype="bf16").run().check()


def test_strides_and_rows_that_no_sequence_has():
    rng = np.random.default_rng(25)
    Call(rng, [3, 0, 1], [20, 4, 0], 40, 4, 2, 128, tail=9, q_pad=24).run().check()
    Call(rng, [1, 1], [20, 4], 0, 4, 4, 64, tail=70).run().check()
    Call(rng, [50, 45], [0, 4], 10, 4, 4, 64, tail=70).run().check()


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 35, 50, 33]])
@pytest.mark.parametrize("hd", [64, 512])
def test_pages_with_room_between_them(hd, new):
    """A page stride past the page's rows, NaN between: the same bits."""
    rng = np.random.default_rng(26)
    c = Call(rng, new, [20] * 4, 100, 4, 2, hd)
    near = c.run().out.clone()
    stride = c.pool.stride + 72
    wide = [torch.full((c.pool.npages, stride), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]
    for w, raw in zip(wide, (c.pool.k_raw, c.pool.v_raw)):
        w[:, :c.pool.stride] = raw
    c.kv = g.PagedKv(wide[0].data_ptr(), wide[1].data_ptr(), c.pool.npages, 2, c.pool.page, hd, g.ELEM_F16, stride)
    c.out.fill_(5.0)
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(near, c.out)


def test_two_sequences_on_the_same_pages():
    """Forks of one sequence: the same rows under two numbers, other queries."""
    rng = np.random.default_rng(28)
    c = Call(rng, [1, 1, 1], [49, 49, 30], 64, 4, 2, 128)
    c.pool.table[1] = c.pool.table[0]
    c.pool.table_host[1] = c.pool.table_host[0]
    c.run().check()


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 35, 50, 33], [2, 5, 1, 3]])
def test_tokens_that_see_nothing(new):
    """No prefix and lengths too short for the tokens: zeros and -infinity."""
    rng = np.random.default_rng(27)
    c = Call(rng, new, [20] * 4, 0, 4, 2, 64)
    short = c.pool.lens_host.copy()
    short[1], short[2] = 0, new[2] // 2
    c.pool.lens.copy_(torch.from_numpy(short))
    c.run()
    torch.cuda.synchronize()
    at = np.concatenate([[0], np.cumsum(new)])
    empty = torch.zeros(c.t, dtype=torch.bool)
    empty[at[1]:at[2]] = True
    empty[at[2]:at[3] - new[2] // 2] = True
    out, lse = c.out[:, :256].cpu(), c.lse.cpu()
    assert bool((out[empty] == 0).all()) and bool((lse[empty] == -np.inf).all())
    assert bool(torch.isfinite(lse[~empty]).all()) and bool(out[~empty].abs().sum(-1).gt(0).all())


@pytest.mark.parametrize("new", [[1] * 5, [33, 40, 36, 47, 50], [3, 1, 2, 4, 1]])
@pytest.mark.parametrize("hd", [64, 256, 512])
def test_what_unseen_rows_hold_does_not_matter(hd, new):
    """NaN and infinities on pages nobody has, behind every sequence's last row and behind the prefix."""
    rng = np.random.default_rng(29)
    c = Call(rng, new, [0, 17, 30, 15, 40], 77, 4, 2, hd, page=32, dtype="bf16", spare=4)
    seen = torch.zeros(c.pool.npages, c.pool.page, dtype=torch.bool)
    for s, n in enumerate(c.pool.lens_host):
        r = np.arange(n)
        seen[torch.from_numpy(c.pool.table_host[s, r // 32].astype(np.int64)), torch.from_numpy(r % 32)] = True
    r = np.arange(77)
    seen[torch.from_numpy(c.pool.prefix_ids[r // 32].astype(np.int64)), torch.from_numpy(r % 32)] = True
    junk = torch.tensor([float("nan"), float("inf"), -float("inf")])[torch.randint(3, (c.pool.npages, 1, 32, 1))]
    for x in (c.pool.k, c.pool.v):
        x.copy_(torch.where(seen[:, None, :, None].cuda(), x, junk.to(x.dtype).cuda()))
    # (the plain form reads the seen rows alone)
    c.run().check()


@pytest.mark.parametrize("window", [0, 25])
@pytest.mark.parametrize("new,before", [([1] * 7, 0), ([33, 40, 36, 47, 50], 0), ([3, 1, 2, 4, 1], 0), ([1] * 3, 900),
                                        ([40, 60, 35], 700)])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_nan_reaches_the_queries_that_see_its_row_and_no_others(hd, new, before, window):
    """One sequence's values NaN in a row that some of its queries see, then
    keys; the rest of its queries and the other sequences are as without it."""
    rng = np.random.default_rng(30)
    c = Call(rng, new, before + np.array([0, 17, 30, 15, 40, 31, 47])[:len(new)], 77, 4, 2, hd, page=32, dtype="bf16",
             window=window)
    clean = c.run().out.clone(), c.lse.clone()
    c.check("clean")
    s = 1
    n, length = new[s], int(c.pool.lens_host[s])
    row = length - max(1, n // 2)  # the last half of its queries see it
    own = length - n + np.arange(n)
    sees = (own >= row) & ((own < row + window) if window else True)
    if before or n == 1:  # a row of the first tile, behind the window where there is one
        row = max(0, length - n - 1 - (30 if window else 0))
        sees = np.full(n, True) if not window else (own < row + window)
    at = int(np.sum(new[:s])) + np.flatnonzero(sees)
    for raw in (c.pool.v, c.pool.k):
        old = raw.clone()
        raw[int(c.pool.table_host[s, row // 32]), :, row % 32] = float("nan")
        c.out.fill_(5.0)
        c.lse.fill_(5.0)
        c.run()
        torch.cuda.synchronize()
        assert bool(torch.isnan(c.out[at, :4 * hd]).all())
        c.out[at], c.lse[at] = clean[0][at], clean[1][at]
        raw.copy_(old)
        c.check("NaN in a row")


@pytest.mark.parametrize("new", [[1] * 7, [33, 40, 36, 47, 50], [3, 1, 2, 4, 1]])
@pytest.mark.parametrize("hd", [64, 256, 512])
def test_a_query_of_nan_spoils_its_own_row_alone(hd, new):
    rng = np.random.default_rng(32)
    c = Call(rng, new, [20] * len(new), 300, 4, 2, hd)
    clean = c.run().out.clone(), c.lse.clone()
    c.q[2, hd:2 * hd] = float("nan")  # (token 2, head 1)
    c.q[2, 3 * hd] = float("inf")     # (head 3: scores of both signs, infinite)
    c.out.fill_(5.0)
    c.run()
    torch.cuda.synchronize()
    mine = torch.zeros(c.rows, 4, hd, dtype=torch.bool, device="cuda")
    mine[2, 1], mine[2, 3] = True, True
    mine = mine.view(c.rows, 4 * hd)
    assert bool(torch.isnan(c.out[2, hd:2 * hd]).all()) and bool(torch.isnan(c.out[2, 3 * hd:4 * hd]).all())
    assert torch.equal(c.out[:, :4 * hd][~mine], clean[0][:, :4 * hd][~mine])


def test_values_of_infinity_that_a_row_sees():
    """One key's values infinite of both signs, seen by the second half of a question: infinite there, as without them
    before."""
    rng = np.random.default_rng(34)
    for hd, new in ((128, [64, 40]), (256, [4, 3])):
        c = Call(rng, new, [10, 10], 40, 4, 2, hd)
        clean = c.run().out.clone()
        row = 10 + new[0] // 2
        sign = torch.where(torch.arange(hd) % 2 == 0, 1.0, -1.0).half().cuda()
        c.pool.v[int(c.pool.table_host[0, row // 16]), :, row % 16] = sign * float("inf")
        c.run()
        torch.cuda.synchronize()
        at = new[0] // 2
        assert torch.equal(c.out[at:new[0], :4 * hd], (sign * float("inf")).repeat(4).expand(new[0] - at, -1))
        got, exp = torch.cat([c.out[:at], c.out[new[0]:]]), torch.cat([clean[:at], clean[new[0]:]])
        # (one of the two rounds p: 2^-11 of sum p |v|, which is below 6; each output rounds by half a step)
        assert bool(((got - exp).abs().float() <= 2.0 ** -10 * exp.abs().float() + 6 * 2.0 ** -11).all())


def test_pages_outside_the_pool_are_not_seen():
    rng = np.random.default_rng(31)
    for new in ([1] * 4, [35, 40, 50, 33], [3, 4, 1, 2]):
        c = Call(rng, new, [40, 60, 50, 45], 50, 4, 2, 128, page=16)
        c.pool.table[0, 1], c.pool.table[1, 0], c.pool.table[1, 2] = c.pool.npages, -1, 1 << 30
        hidden = {0: [1], 1: [0, 2]}

        def gone(s, n):
            pages = np.arange(n) // 16
            return torch.from_numpy(np.isin(pages, hidden.get(s, [])))

        c.run().check(skip_keys=gone)


def test_lengths_past_the_table_stop_at_its_end():
    rng = np.random.default_rng(33)
    c = Call(rng, [1, 1], [31, 31], 20, 2, 1, 64, page=32)
    whole = c.run().out.clone()
    c.pool.lens[0] = 1000
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(whole, c.out)


def test_pool_past_32_bit_offsets():
    """Pages whose bytes and elements lie past 2^32."""
    rng = np.random.default_rng(35)
    npages, kv_heads, page, hd = 70_000, 2, 128, 256  # 9.2 GB each for k and v
    lens = np.array([150, 129])
    c = Call(rng, [1, 1], lens - 1, 200, 4, kv_heads, hd, page=page)
    big = [torch.zeros(npages, kv_heads, page, hd, dtype=torch.float16, device="cuda") for _ in range(2)]
    place = rng.choice(np.arange(npages - 3000, npages), c.pool.npages, replace=False)
    for b, x in zip(big, (c.pool.k, c.pool.v)):
        b[torch.from_numpy(place).cuda()] = x
    near = c.run().out.clone()
    place_d = torch.from_numpy(place.astype(np.int32)).cuda()
    c.pool.table.copy_(place_d[c.pool.table.long()])
    c.pool.prefix_table.copy_(place_d[c.pool.prefix_table.long()])
    c.kv = g.PagedKv(big[0].data_ptr(), big[1].data_ptr(), npages, kv_heads, page, hd, g.ELEM_F16)
    c.out.fill_(5.0)
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(near, c.out)


@pytest.mark.parametrize("new", [[1] * 12, [40, 38, 50, 33, 61], [3] * 7])
def test_the_same_call_gives_the_same_bits(new):
    rng = np.random.default_rng(37)
    c = Call(rng, new, [50] * len(new), 900, 4, 1, 256)
    first = c.run().out.clone(), c.lse.clone()
    for _ in range(5):
        c.ws.random_(0, 256)
        c.run()
        torch.cuda.synchronize()
        assert torch.equal(first[0], c.out) and torch.equal(first[1], c.lse)


def test_captured_calls_replay_with_the_lengths_of_the_moment():
    rng = np.random.default_rng(39)
    c = Call(rng, [1] * 6, [199] * 6, 100, 4, 2, 128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for n in (1, 17, 200, 64):
        c.pool.lens.fill_(n)
        c.q.normal_()
        c.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = c.out.clone(), c.lse.clone()
        c.out.zero_()
        c.run()
        torch.cuda.synchronize()
        assert torch.equal(got[0][:, :512], c.out[:, :512]) and torch.equal(got[1], c.lse)


def test_calls_on_two_streams():
    rng = np.random.default_rng(41)
    calls = [Call(rng, [1] * 30, rng.integers(0, 500, 30), 2000, 8, 4, 256) for _ in range(2)]
    for c in calls:
        c.exp = c.run().out.clone()
        c.out.fill_(5.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(4):
        for c, s in zip(calls, streams):
            c.run(s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        assert torch.equal(c.out, c.exp)


def test_large_scores_and_infinite_ones():
    """Scores of hundreds in a row's early keys and late ones; one key whose score is -infinity."""
    rng = np.random.default_rng(43)
    Call(rng, [1] * 4, [200] * 4, 500, 4, 1, 256, qscale=60.0).run().check()
    Call(rng, [40] * 4, [20] * 4, 500, 4, 1, 64, qscale=60.0, dtype="bf16").run().check()


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 33, 50], [2, 1, 3]])
def test_many_small_probabilities_beside_a_large_one(new):
    """60,000 shared keys whose probabilities are 2^-20.5 of one own key's: 4 % of the sum, all of the output."""
    rng = np.random.default_rng(47)
    c = Call(rng, new, [20] * 3, 60_000, 2, 1, 64, page=64)
    c.q.fill_(1.0)
    c.pool.k.zero_()
    c.pool.v.fill_(1.0)
    for s in range(3):
        page = int(c.pool.table_host[s, 0])
        c.pool.k[page, 0, 0] = 14.25 * 8 / 64  # (its score is 14.25: e^-14.25 = 2^-20.6)
        c.pool.v[page, 0, 0] = 0.0
    c.run().check()


@pytest.mark.parametrize("new", [[0, 5, 0, 0, 7, 1, 0], [0, 50, 0, 130, 0], [0, 0, 1]])
def test_sequences_without_new_tokens(new):
    rng = np.random.default_rng(49)
    c = Call(rng, new, rng.integers(0, 90, len(new)), 100, 8, 2, 128, single=False)
    c.run().check()


def test_refuses_a_short_workspace():
    c = Call(np.random.default_rng(45), [1] * 4, [5] * 4, 3000, 4, 1, 256)
    assert c.ws.numel() > 0
    c.ws = c.ws[:-16]
    with pytest.raises(g.OmgError, match="workspace needs"):
        c.run()


BATCHES = [([1] * 7, [20] * 7, 300), ([1] * 70, [90] * 70, 301), ([33, 40, 36, 47, 50], [0, 17, 30, 15, 40], 200),
           ([3, 1, 2, 4, 1], [9, 0, 200, 4, 31], 77), ([50] * 45, [5] * 45, 70), ([9, 70], [400, 700], 0)]


@pytest.mark.parametrize("new,before,prefix", BATCHES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_values_up_to_the_types_largest(hd, new, before, prefix):
    """bf16 values of up to 3e38: sums over keys, unlike their mean, lie past f32's largest."""
    rng = np.random.default_rng(51 + hd)
    c = Call(rng, new, before, prefix, 16 if len(new) == 45 else 4, 8 if len(new) == 45 else 2, hd, dtype="bf16")
    c.pool.v_raw.copy_((c.pool.v_raw.float() * 1e38).clamp_(-3e38, 3e38))
    c.run().check()


@pytest.mark.parametrize("new,before,prefix", BATCHES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_equal_values_up_to_the_types_largest(hd, dtype, new, before, prefix):
    """All keys' values alike, the type's largest among them: their mean within the probabilities' rounding, and finite."""
    rng = np.random.default_rng(53 + hd)
    c = Call(rng, new, before, prefix, 16 if len(new) == 45 else 4, 8 if len(new) == 45 else 2, hd, dtype=dtype)
    most = torch.finfo(TYPES[dtype]).max
    row = torch.randn(hd).to(TYPES[dtype])
    row[::5], row[1::5] = most, -most
    c.pool.v.copy_(row.cuda())
    c.run().check()
    assert bool(torch.isfinite(c.out).all())


@pytest.mark.parametrize("new", [[1] * 4, [40, 35, 50, 33], [6, 5, 9, 7]])
def test_the_largest_window_is_no_window(new):
    """A window of 2^31 - 1, with sequences whose lengths are short of their tokens: positions below zero."""
    rng = np.random.default_rng(55)
    c = Call(rng, new, [0, 20, 3, 0], 2, 4, 2, 64)
    c.pool.lens.copy_(torch.tensor([max(0, new[0] - 6), new[1] + 20, new[2] // 2, 0], dtype=torch.int32))
    c.run()
    torch.cuda.synchronize()
    whole = c.out.clone(), c.lse.clone()
    c.window = 2 ** 31 - 1
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(whole[0], c.out) and torch.equal(whole[1], c.lse)


@pytest.mark.parametrize("new,heads", [([1], 4), ([1, 1], 2), ([5], 2)])
def test_the_most_splits_of_prefix_and_own_rows(new, heads):
    """64 splits each: a join of 128 partial results."""
    rng = np.random.default_rng(57)
    Call(rng, new, [9000] * len(new), 5000, heads, 1, 128, page=64).run().check()
    Call(rng, new, [9000] * len(new), 5000, heads, 1, 128, page=64, window=9700, dtype="bf16").run().check()
