"""The calls for long caches as a program runs them together, each step also
captured and replayed: drafts verified as trees and their accepted paths closed
up; attention weights gathered and the cache cut by them when it is full; a step
over the few blocks that the pages' means choose.

The model is one attention layer whose projections are a table, a row of qkv
per token id; which token follows is given.  Tolerance of the attention's
outputs against 64 bits: as in the token-by-token test (one rounding of q, k, v,
p and the output each, f32 rotations and sums); cached rows are compared bit for
bit with those that appending token by token leaves."""
from __future__ import annotations

import numpy as np
import pytest

import grande_amd as g
from paged import ELEM, TYPES, half_step, rope_table

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

VOCAB = 300


def i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def rotated(x, cs):
    """[..., hd] by (cos, sin) pairs [..., hd / 2][2], pairs (i, i + hd / 2)."""
    a, b = x.chunk(2, -1)
    c, s = cs[..., 0], cs[..., 1]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def stream():
    return torch.cuda.current_stream().cuda_stream


class Layer:
    """Pages of `nseq` sequences of up to `most` rows, shared prefix pages, and the layer's projections."""

    def __init__(self, seed, nseq, prefix, most, heads, kv_heads, hd, dtype, page=16, spare=0):
        rng = np.random.default_rng(seed)
        self.rng, self.nseq, self.prefix, self.heads, self.kv_heads, self.hd = rng, nseq, prefix, heads, kv_heads, hd
        self.dtype, self.page, self.width = dtype, page, (heads + 2 * kv_heads) * hd
        self.qkv_of = torch.from_numpy(rng.standard_normal((VOCAB, self.width)).astype(np.float32)).cuda()
        self.max_pages, pre = -(-most // page), -(-prefix // page)
        ids = rng.permutation(pre + nseq * (self.max_pages + spare)).astype(np.int32)
        self.prefix_table = i32(ids[:max(pre, 1)])
        self.table = i32(ids[pre:pre + nseq * self.max_pages].reshape(nseq, -1))
        self.spare = i32(ids[pre + nseq * self.max_pages:].reshape(nseq, -1)) if spare else None
        self.k, self.v = (torch.full((len(ids), kv_heads, page, hd), float("nan"), device="cuda").to(TYPES[dtype])
                          for _ in range(2))
        self.kv = g.PagedKv(self.k.data_ptr(), self.v.data_ptr(), len(ids), kv_heads, page, hd, ELEM[dtype])
        self.rope = rope_table(prefix + most + 64, hd).cuda()
        self.lens = torch.zeros(nseq, dtype=torch.int32, device="cuda")
        self.scale = hd ** -0.5

    def batch(self, tokens, start=None, table=None):
        t = self.table if table is None else table
        return g.PagedBatch(self.nseq, tokens, self.lens.data_ptr(), t.data_ptr(), t.shape[1],
                            start.data_ptr() if start is not None else None, self.prefix_table.data_ptr(), self.prefix)

    def append(self, batch, ids, q, positions=None):
        self.qkv = self.qkv_of.index_select(0, ids)  # (read when the stream runs: kept)
        x, size = self.qkv.data_ptr(), 4
        self.kv.append(batch, g.KvSource(g.ELEM_F32, self.heads, x, x + self.heads * self.hd * size,
                                         x + (self.heads + self.kv_heads) * self.hd * size, self.width,
                                         rope=self.rope.data_ptr(), rope_rows=self.rope.shape[0], rope_dims=self.hd,
                                         positions=positions.data_ptr() if positions is not None else None),
                       q.data_ptr(), self.heads * self.hd, stream())

    def room(self, n):
        return torch.full((n + 16,), 0xFF, dtype=torch.uint8, device="cuda")

    def read_prefix(self, ids):
        n, start = i32([self.prefix]), i32([0, self.prefix])
        b = g.PagedBatch(1, self.prefix, n.data_ptr(), self.prefix_table.data_ptr(), self.prefix_table.numel(), start.data_ptr())
        q = torch.empty(self.prefix, self.heads * self.hd, dtype=TYPES[self.dtype], device="cuda")
        self.append(b, torch.from_numpy(ids).cuda(), q)
        torch.cuda.synchronize()
        return b, n, start

    def own_rows(self, x, s, n, table=None):
        t = (self.table if table is None else table).cpu().numpy()
        r = np.arange(n)
        return x.cpu()[torch.from_numpy(t[s, r // self.page].astype(np.int64)), :, torch.from_numpy(r % self.page)]

    def attend(self, ids, positions, q_id, q_pos, see):
        """One query (token id, position) over keys (ids, positions) that `see` leaves, per KV head a mask
        [kv_heads][keys]: the output, its tolerance and the probabilities, in 64 bits."""
        H, K, D = self.heads, self.kv_heads, self.hd
        x, cs = self.qkv_of.double().cpu(), self.rope.double().cpu()
        qr = rotated(x[q_id].view(-1, D)[:H], cs[q_pos])
        kv = x[torch.from_numpy(np.asarray(ids))].view(len(ids), H + 2 * K, D)
        k = rotated(kv[:, H:H + K], cs[torch.from_numpy(np.asarray(positions))][:, None])
        h = half_step(TYPES[self.dtype])
        out, tol, ps = torch.empty(H, D, dtype=torch.float64), torch.empty(H, D, dtype=torch.float64), []
        for i in range(H):
            m = torch.from_numpy(see[i // (H // K)])
            kh, vh = k[:, i // (H // K)], kv[:, H + K + i // (H // K)]
            p = ((kh @ qr[i]) * self.scale).masked_fill(~m, -np.inf).softmax(-1)
            d = (2 * h + h * h + 2.0 ** -16) * (kh.abs() @ qr[i].abs() * self.scale).masked_fill(~m, 0).max()
            out[i], tol[i] = p @ vh, (p @ vh.abs()) * (torch.expm1(2 * d) + 3 * h + 2.0 ** -17)
            ps.append((p, torch.expm1(2 * d)))
        return out.reshape(-1), tol.reshape(-1), ps


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd,dtype,window", [(4, 1, 256, "bf16", 0), (15, 5, 64, "f16", 0), (8, 2, 128, "f16", 25)])
def test_drafts_verified_as_trees(heads, kv_heads, hd, dtype, window, captured):
    """Every step appends a tree of 11 drafts a sequence with the tokens that do
    follow somewhere in it, attends, and closes up the accepted path.  At the
    end the cache holds what appending token by token leaves."""
    nseq, prefix, N, STEPS = 4, 45, 11, 5
    m = Layer(7 + hd, nseq, prefix, 100, heads, kv_heads, hd, dtype)
    rng = m.rng
    prompt = rng.integers(0, VOCAB, prefix)
    m.read_prefix(prompt)
    truth = rng.integers(0, VOCAB, (nseq, 60))
    have = np.zeros(nseq, int)
    t = nseq * N
    start = i32(np.arange(nseq + 1) * N)
    q, out = (torch.empty(t, heads * hd, dtype=TYPES[dtype], device="cuda") for _ in range(2))
    ids, positions = torch.zeros(t, dtype=torch.int64, device="cuda"), i32(np.zeros(t))
    mask, base, rows = i32(np.zeros((t, 1))), i32(np.zeros(nseq)), i32(np.full((nseq, N), -1))
    b = m.batch(t, start)
    ws = m.room(m.kv.attention_tree_workspace(b, heads))

    def verify():
        m.lens.add_(N)
        m.append(b, ids, q, positions)
        m.kv.attention_tree(b, heads, q.data_ptr(), heads * hd, out.data_ptr(), heads * hd, m.scale, mask.data_ptr(), 1,
                            window=window, positions=positions.data_ptr(), workspace=ws.data_ptr(),
                            workspace_bytes=ws.numel(), stream=stream())

    def accept():
        m.kv.keep(b, rows.data_ptr(), N, N, first=base.data_ptr(), stream=stream())
        m.lens.copy_(base + (rows >= 0).sum(1))

    graphs = []
    if captured:
        side = torch.cuda.Stream()  # the libraries' first calls, outside the capture
        with torch.cuda.stream(side):
            verify(), accept()
        side.synchronize()
        for f in (verify, accept):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                f()
    m.lens.zero_()
    for step in range(STEPS):
        draft, see, depth, paths = np.zeros((nseq, N), int), np.zeros((nseq, N, N), bool), np.zeros((nseq, N), int), []
        for s in range(nseq):
            good = int(rng.integers(1, 6))  # so many tokens of the truth lie in the tree
            path = np.sort(rng.permutation(N)[:good])
            draft[s] = rng.integers(0, VOCAB, N)
            for i in range(N):
                on = np.flatnonzero(path == i)
                parent = (path[on[0] - 1] if on[0] else -1) if len(on) else int(rng.integers(-1, i)) if i else -1
                if parent >= 0:
                    see[s, i], depth[s, i] = see[s, parent], depth[s, parent] + 1
                see[s, i, i] = True
                if len(on):
                    draft[s, i] = truth[s, have[s] + on[0]]
            paths.append(path)
        bits = (see.reshape(t, N) * (1 << np.arange(N))).sum(1)
        at = prefix + have[:, None] + depth
        ids.copy_(torch.from_numpy(draft.reshape(-1)))
        positions.copy_(i32(at.reshape(-1)))
        mask.copy_(i32(bits[:, None]))
        base.copy_(i32(have))
        graphs[0].replay() if captured else verify()
        torch.cuda.synchronize()
        for s in range(nseq):
            keys = np.concatenate([prompt, truth[s, :have[s]], draft[s]])
            key_at = np.concatenate([np.arange(prefix + have[s]), at[s]])
            for i in range(N):
                m_ = np.concatenate([np.ones(prefix + have[s], bool), see[s, i]])
                if window:
                    m_[:prefix + have[s]] &= at[s, i] - np.arange(prefix + have[s]) < window
                exp, tol, _ = m.attend(keys, key_at, draft[s, i], at[s, i], np.tile(m_, (kv_heads, 1)))
                off = (out[s * N + i].double().cpu() - exp).abs() - tol
                assert bool((off <= 0).all()), f"step {step} sequence {s} draft {i}: {float(off.max())}"
        r = np.full((nseq, N), -1)
        for s, path in enumerate(paths):
            r[s, :len(path)] = have[s] + path
            have[s] += len(path)
        rows.copy_(i32(r))
        graphs[1].replay() if captured else accept()
        torch.cuda.synchronize()
        assert np.array_equal(m.lens.cpu().numpy(), have)
    # token by token on the same pages
    for s in range(nseq):
        got = [m.own_rows(x, s, have[s]) for x in (m.k, m.v)]
        m.lens.copy_(i32(have))
        st = i32([0, have[s]])
        one = g.PagedBatch(1, int(have[s]), m.lens[s:].data_ptr(), m.table[s].data_ptr(), m.max_pages, st.data_ptr(),
                           m.prefix_table.data_ptr(), prefix)
        m.append(one, torch.from_numpy(truth[s, :have[s]]).cuda(), torch.empty(int(have[s]), heads * hd, dtype=TYPES[dtype], device="cuda"))
        torch.cuda.synchronize()
        for a, x in zip(got, (m.k, m.v)):
            assert torch.equal(a.view(torch.int16), m.own_rows(x, s, have[s]).view(torch.int16)), f"sequence {s}"


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd,dtype,apart", [(4, 1, 256, "bf16", False), (15, 5, 64, "f16", True), (8, 2, 128, "f16", False)])
def test_a_cache_cut_by_its_weights(heads, kv_heads, hd, dtype, apart, captured):
    """Decoding with a budget: each step attends, gathers its weights, and cuts
    every sequence back to KEEP rows; what a head keeps is what its weights say,
    and later steps attend over that."""
    nseq, prefix, KEEP, RECENT, STEPS, BEFORE = 3, 20, 24, 6, 9, 21
    m = Layer(50 + hd, nseq, prefix, 48, heads, kv_heads, hd, dtype, spare=3 if apart else 0)
    rng = m.rng
    prompt, text = rng.integers(0, VOCAB, prefix), rng.integers(0, VOCAB, (nseq, BEFORE + STEPS))
    m.read_prefix(prompt)
    ldw = m.max_pages * m.page
    w = torch.zeros(nseq, kv_heads, ldw, device="cuda")
    w_next = torch.zeros_like(w)
    rows = torch.zeros(nseq, kv_heads, KEEP, dtype=torch.int32, device="cuda")
    q, out = (torch.empty(nseq, heads * hd, dtype=TYPES[dtype], device="cuda") for _ in range(2))
    lse, ids, positions = torch.zeros(nseq, heads, device="cuda"), torch.zeros(nseq, dtype=torch.int64, device="cuda"), i32(np.zeros(nseq))
    b = m.batch(nseq)
    ws = m.room(m.kv.attention_workspace(b, heads))
    ws_w = m.room(m.kv.attention_weights_workspace(b, heads))

    def step():
        m.lens.add_(1)
        m.append(b, ids, q, positions)
        m.kv.attention(b, heads, q.data_ptr(), heads * hd, out.data_ptr(), heads * hd, m.scale, lse=lse.data_ptr(),
                       workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=stream())
        m.kv.attention_weights(b, heads, q.data_ptr(), heads * hd, lse.data_ptr(), m.scale, w.data_ptr(), ldw,
                               workspace=ws_w.data_ptr(), workspace_bytes=ws_w.numel(), stream=stream())

    def cut():
        if not apart:
            m.kv.evict(b, KEEP, RECENT, w.data_ptr(), ldw, rows.data_ptr(), stream=stream())
        else:  # to the spare pages and, to go on with the same tables, back: whole lists, each in its order
            m.kv.evict(b, KEEP, RECENT, w.data_ptr(), ldw, rows.data_ptr(), kept_weights=w_next.data_ptr(), kept_ld=ldw,
                       to_table=m.spare.data_ptr(), to_ld=m.spare.shape[1], stream=stream())
            w.copy_(w_next)
            m.kv.keep(m.batch(nseq, table=m.spare), every.data_ptr(), KEEP, KEEP, to_table=m.table.data_ptr(),
                      to_ld=m.max_pages, stream=stream())
            w_next.zero_()
        m.lens.clamp_(max=KEEP)

    every = i32(np.tile(np.arange(KEEP), (nseq, 1)))
    if apart:  # (rows that are not there move as they are)
        m.k.nan_to_num_(), m.v.nan_to_num_()
    # the sequences' first rows, one by one
    kept = [[list(range(BEFORE)) for _ in range(kv_heads)] for _ in range(nseq)]
    weight = np.zeros((nseq, kv_heads, BEFORE + STEPS))
    slack = np.zeros_like(weight)
    start = i32(np.arange(nseq + 1) * BEFORE)
    m.lens.fill_(BEFORE)
    m.append(m.batch(nseq * BEFORE, start), torch.from_numpy(text[:, :BEFORE].reshape(-1)).cuda(),
             torch.empty(nseq * BEFORE, heads * hd, dtype=TYPES[dtype], device="cuda"))
    torch.cuda.synchronize()
    graphs = []
    if captured:
        k, v, lens = m.k.clone(), m.v.clone(), m.lens.clone()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step(), cut()
        side.synchronize()
        for f in (step, cut):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                f()
        m.k.copy_(k), m.v.copy_(v), m.lens.copy_(lens), w.zero_()
    for n in range(STEPS):
        at = BEFORE + n
        ids.copy_(torch.from_numpy(text[:, at]))
        positions.fill_(prefix + at)
        graphs[0].replay() if captured else step()
        torch.cuda.synchronize()
        gathered = w.double().cpu().numpy()
        for s in range(nseq):
            keys = np.concatenate([prompt, text[s, :at + 1]])
            see = np.zeros((kv_heads, prefix + at + 1), bool)
            see[:, :prefix] = True
            for h in range(kv_heads):
                kept[s][h].append(at)
                see[h, prefix + np.asarray(kept[s][h])] = True
            exp, tol, ps = m.attend(keys, np.arange(prefix + at + 1), text[s, at], prefix + at, see)
            off = (out[s].double().cpu() - exp).abs() - tol
            assert bool((off <= 0).all()), f"step {n} sequence {s}: {float(off.max())}"
            for i, (p, d) in enumerate(ps):
                h = i // (heads // kv_heads)
                weight[s, h, :at + 1] += p[prefix:].numpy()
                slack[s, h, :at + 1] += (p[prefix:] * (d + 2.0 ** -15)).numpy()
            for h in range(kv_heads):
                r = np.asarray(kept[s][h])
                off = np.abs(gathered[s, h, :len(r)] - weight[s, h, r]) - slack[s, h, r] - 1e-7
                assert (off <= 0).all(), f"weights, step {n} sequence {s} head {h}"
                assert (gathered[s, h, len(r):] == 0).all()
        graphs[1].replay() if captured else cut()
        torch.cuda.synchronize()
        got = rows.cpu().numpy()
        for s in range(nseq):
            for h in range(kv_heads):
                r = np.asarray(kept[s][h])
                if len(r) > KEEP:
                    old = len(r) - RECENT
                    take = np.sort(np.lexsort((np.arange(old), -gathered[s, h, :old]))[:KEEP - RECENT])
                    take = np.concatenate([take, np.arange(old, len(r))])
                else:
                    take = np.arange(len(r))
                assert np.array_equal(got[s, h, :len(take)], take) and (got[s, h, len(take):] == -1).all()
                kept[s][h] = r[take].tolist()
        assert int(m.lens.max()) <= KEEP


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd,dtype", [(4, 1, 256, "bf16"), (15, 5, 64, "f16"), (8, 2, 128, "f16")])
def test_steps_over_chosen_blocks(heads, kv_heads, hd, dtype, captured):
    """Means kept up by one call behind each append; each step over 4 of the 8
    and more blocks that there are."""
    nseq, prefix, BLOCKS, STEPS, BEFORE = 3, 120, 4, 20, 9
    m = Layer(90 + hd, nseq, prefix, 48, heads, kv_heads, hd, dtype)
    rng = m.rng
    prompt, text = rng.integers(0, VOCAB, prefix), rng.integers(0, VOCAB, (nseq, BEFORE + STEPS))
    means = torch.full((m.k.shape[0], kv_heads, hd), float("nan"), device="cuda")
    pre, *held = m.read_prefix(prompt)
    m.kv.block_means(pre, means.data_ptr(), stream())
    start = i32(np.arange(nseq + 1) * BEFORE)
    m.lens.fill_(BEFORE)
    first = m.batch(nseq * BEFORE, start)
    m.append(first, torch.from_numpy(text[:, :BEFORE].reshape(-1)).cuda(),
             torch.empty(nseq * BEFORE, heads * hd, dtype=TYPES[dtype], device="cuda"))
    m.kv.block_means(first, means.data_ptr(), stream())
    torch.cuda.synchronize()
    q, out = (torch.empty(nseq, heads * hd, dtype=TYPES[dtype], device="cuda") for _ in range(2))
    ids, chosen = torch.zeros(nseq, dtype=torch.int64, device="cuda"), i32(np.zeros((nseq, kv_heads, BLOCKS)))
    b = m.batch(nseq)
    ws = m.room(m.kv.attention_blocks_workspace(b, heads, BLOCKS))

    def step():
        m.lens.add_(1)
        m.append(b, ids, q)
        m.kv.block_means(b, means.data_ptr(), stream())
        m.kv.attention_blocks(b, heads, q.data_ptr(), heads * hd, out.data_ptr(), heads * hd, m.scale, means.data_ptr(),
                              BLOCKS, chosen=chosen.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                              stream=stream())

    if captured:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        m.lens.fill_(BEFORE)
    page, np_ = m.page, -(-prefix // m.page)
    for n in range(STEPS):
        at = BEFORE + n
        ids.copy_(torch.from_numpy(text[:, at]))
        graph.replay() if captured else step()
        torch.cuda.synchronize()
        mean = means.double().cpu()
        for s in range(nseq):
            last = np_ + at // page
            pages = np.concatenate([m.prefix_table.cpu().numpy()[:np_], m.table.cpu().numpy()[s]])[:last + 1].astype(np.int64)
            own = m.own_rows(m.k, s, at + 1).double()[at // page * page:].mean(0)
            assert bool(((mean[pages[-1]] - own).abs() <= 2.0 ** -24 * own.abs()).all())
            qs = q[s].double().cpu().view(kv_heads, heads // kv_heads, hd).sum(1)
            see = np.zeros((kv_heads, prefix + at + 1), bool)
            for h in range(kv_heads):
                score = (mean[pages[:last], h] @ qs[h]).float().numpy()
                take = np.append(np.sort(np.lexsort((np.arange(last), -score))[:BLOCKS - 1]), last)
                assert np.array_equal(chosen[s, h].cpu().numpy(), take), f"step {n} sequence {s} head {h}"
                for blk in take:
                    lo = blk * page if blk < np_ else prefix + (blk - np_) * page
                    see[h, lo:min(lo + page, prefix if blk < np_ else prefix + at + 1)] = True
            exp, tol, _ = m.attend(np.concatenate([prompt, text[s, :at + 1]]), np.arange(prefix + at + 1), text[s, at], prefix + at, see)
            off = (out[s].double().cpu() - exp).abs() - tol
            assert bool((off <= 0).all()), f"step {n} sequence {s}: {float(off.max())}"
