"""omg_dev_kv_append (PagedKv.append) against the plain form in 64 bits:
norms, the three rotation layouts, ragged batches, pages, strides, types,
rows that belong to nobody, and what the call refuses.

Tolerance: one rounding to the cache's type is at most half a step of the
value; the f32 arithmetic before it (a sum of at most 512 squares, a square
root, four products and a sum) stays below 2^-18 of the head's largest
rotated pair."""
from __future__ import annotations

import numpy as np
import pytest

import grande_amd as g
from paged import ELEM, TYPES, Pool, half_step, plain_norm, plain_rope, rope_table, starts

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = 1e-6


def close(got, exp, dtype, what):
    """Within one rounding of the type plus 2^-18 of the row's largest value."""
    got, exp = got.double().cpu(), exp.double()
    tol = half_step(dtype) * exp.abs() + 2.0 ** -18 * exp.abs().amax(-1, keepdim=True) + 1e-7
    bad = (got - exp).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((got - exp).abs().max())}"


def run_append(rng, new, before, heads, kv_heads, hd, page, src, dtype, layout, dims, norms, prefix=0, pad=0,
               page_pad=0, tail=0, positions=False):
    """One append of `new` tokens per sequence after `before` rows; checks
    queries, the appended rows and that nothing else changed."""
    new, before = np.asarray(new), np.asarray(before)
    pool = Pool(rng, new + before, prefix, kv_heads, hd, page, dtype, page_pad=page_pad)
    t = int(new.sum())
    rows = t + tail
    ld = (heads + 2 * kv_heads) * hd + pad
    qkv = torch.from_numpy(rng.standard_normal((rows, ld)).astype(np.float32)).to(TYPES[src]).cuda()
    table = rope_table(int((new + before).max()) + prefix, dims).cuda() if dims else None
    qn, kn = (torch.from_numpy((1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)).cuda() for _ in range(2))
    q_out = torch.full((rows, heads * hd + 8), 7.0, dtype=TYPES[dtype], device="cuda")
    pos_host = np.concatenate([prefix + b + np.arange(n) for n, b in zip(new, before)])
    if positions:
        pos_host = rng.permutation(pos_host) - 3  # some below the table's first row
    pos = torch.from_numpy(pos_host.astype(np.int32)).cuda() if positions else None
    x, size = qkv.data_ptr(), qkv.element_size()
    k0, v0 = pool.k_raw.clone(), pool.v_raw.clone()
    single = bool((new == 1).all()) and tail == 0
    start = None if single else starts(new)
    s = g.KvSource(ELEM[src], heads, x, x + heads * hd * size, x + (heads + kv_heads) * hd * size, ld,
                   rope=table.data_ptr() if dims else None, rope_rows=table.shape[0] if dims else 0, rope_dims=dims,
                   rope_layout=layout, positions=pos.data_ptr() if positions else None,
                   q_norm=qn.data_ptr() if norms else None, k_norm=kn.data_ptr() if norms else None, v_norm=norms,
                   eps=EPS, q_scale=0.25)
    pool.kv().append(pool.batch(rows, start), s, q_out.data_ptr(), heads * hd + 8)
    torch.cuda.synchronize()

    xf = qkv.double().cpu()[:t, :(heads + 2 * kv_heads) * hd].view(t, -1, hd)
    q, k, v = xf[:, :heads], xf[:, heads:heads + kv_heads], xf[:, heads + kv_heads:]
    if norms:
        q, k, v = plain_norm(q, qn, EPS), plain_norm(k, kn, EPS), plain_norm(v, None, EPS)
    if dims:
        cs = table.cpu()[np.clip(pos_host, 0, table.shape[0] - 1)]
        q, k = (torch.stack([plain_rope(y[i], cs[i], layout) for i in range(t)]) for y in (q, k))
    close(q_out[:t, :heads * hd].reshape(t, heads, hd), q * 0.25, TYPES[dtype], "q")
    assert bool((q_out[:, heads * hd:] == 7.0).all()) and bool((q_out[t:] == 7.0).all())
    touched = torch.zeros(pool.npages, page, dtype=torch.bool)
    at = 0
    for i, (n, b) in enumerate(zip(new, before)):
        r = b + np.arange(n)
        p, o = torch.from_numpy(pool.table_host[i, r // page].astype(np.int64)), torch.from_numpy(r % page)
        close(pool.k.cpu()[p, :, o], k[at:at + n], TYPES[dtype], f"k of sequence {i}")
        close(pool.v.cpu()[p, :, o], v[at:at + n], TYPES[dtype], f"v of sequence {i}")
        touched[p, o] = True
        at += n
    for now, old in ((pool.k, pool.view(k0)), (pool.v, pool.view(v0))):
        same = (now == old).permute(0, 2, 1, 3).flatten(2).all(-1).cpu()
        assert bool(same[~touched].all()), "rows that no token names changed"
    if page_pad:
        n = kv_heads * page * hd
        assert torch.equal(pool.k_raw[:, n:], k0[:, n:]) and torch.equal(pool.v_raw[:, n:], v0[:, n:])


@pytest.mark.parametrize("layout", [g.ROPE_HALF, g.ROPE_INTERLEAVED, g.ROPE_HEAD_HALF])
@pytest.mark.parametrize("hd,dims", [(64, 64), (64, 16), (128, 32), (128, 96), (256, 256), (256, 64), (512, 128),
                                     (512, 512)])
def test_layouts_and_widths(hd, dims, layout):
    rng = np.random.default_rng(hd * 7 + dims + layout)
    run_append(rng, [3, 1, 7], [0, 15, 30], 4, 2, hd, 16, "f32", "f16", layout, dims, True)


@pytest.mark.parametrize("src,dtype", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 1, 256), (15, 5, 64), (1, 1, 128), (8, 1, 512), (28, 4, 128)])
def test_types_and_head_counts(src, dtype, heads, kv_heads, hd):
    rng = np.random.default_rng(heads * 31 + hd)
    run_append(rng, [1] * 9, np.arange(9) * 5, heads, kv_heads, hd, 32, src, dtype, g.ROPE_HALF, hd, heads != 15)


def test_long_ragged_prompts_over_many_sequences():
    rng = np.random.default_rng(3)
    new = np.array([700, 1, 0, 333, 64, 0, 129])  # two sequences without a token
    run_append(rng, new, [5, 0, 9, 63, 64, 0, 1], 8, 4, 256, 64, "f32", "f16", g.ROPE_HALF, 256, True, prefix=100)


def test_many_sequences_find_their_rows():
    """5,000 sequences of zero to three tokens: the search takes more than one step."""
    rng = np.random.default_rng(5)
    run_append(rng, rng.integers(0, 4, 5000), rng.integers(0, 20, 5000), 1, 1, 64, 16, "bf16", "bf16",
               g.ROPE_INTERLEAVED, 16, False)


def test_strides_and_rows_that_no_sequence_has():
    rng = np.random.default_rng(7)
    run_append(rng, [2, 5], [14, 1], 3, 3, 128, 16, "f32", "bf16", g.ROPE_HALF, 128, True, pad=24, page_pad=72, tail=6)


def test_positions_of_their_own_are_clamped_to_the_table():
    rng = np.random.default_rng(9)
    run_append(rng, [6, 5], [0, 20], 2, 1, 64, 16, "f32", "f16", g.ROPE_HALF, 64, False, positions=True)


def test_no_rotation_copies_values_of_the_same_type():
    rng = np.random.default_rng(11)
    run_append(rng, [40, 1], [0, 3], 2, 2, 64, 16, "bf16", "bf16", 0, 0, False)


@pytest.mark.parametrize("layout", [g.ROPE_HALF, g.ROPE_INTERLEAVED, g.ROPE_HEAD_HALF])
@pytest.mark.parametrize("dims", [0, 32])
def test_infinities_outside_the_rotation_stay(dims, layout):
    """Elements that no pair holds keep their bits (infinities, NaN beside
    them) and do not reach the rotated ones."""
    rng = np.random.default_rng(12)
    pool = Pool(rng, [5, 9], 0, 2, 128, 16, "f16")
    x = torch.from_numpy(rng.standard_normal((2, 6, 128)).astype(np.float32)).half().cuda()
    pairs = {g.ROPE_HALF: range(dims), g.ROPE_INTERLEAVED: range(dims),
             g.ROPE_HEAD_HALF: [*range(dims // 2), *range(64, 64 + dims // 2)]}[layout]
    out = torch.ones(128, dtype=torch.bool)
    out[list(pairs)] = False
    junk = torch.tensor([float("inf"), -float("inf"), float("nan"), 2.0], dtype=torch.float16).repeat(32).cuda()
    y = torch.where(out.cuda(), junk, x)
    table = rope_table(16, dims).cuda() if dims else None
    q = [torch.zeros(2, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    for src, to in zip((x, y), q):
        at = src.data_ptr()
        pool.kv().append(pool.batch(2), g.KvSource(g.ELEM_F16, 2, at, at + 512, at + 1024, 768,
                                                   rope=table.data_ptr() if dims else None, rope_rows=16 if dims else 0,
                                                   rope_dims=dims, rope_layout=layout), to.data_ptr(), 256)
    torch.cuda.synchronize()
    assert torch.equal(q[0][..., ~out], q[1][..., ~out])
    row = torch.stack([pool.k[int(pool.table_host[s, 0]), :, n - 1] for s, n in enumerate([5, 9])])
    for got in (q[1], row):
        bits = got[..., out].contiguous().view(torch.int16)
        exp = y[:, :2, out].contiguous().view(torch.int16)
        nan = torch.isnan(y[:, :2, out])
        assert torch.equal(bits[~nan], exp[~nan]) and bool(torch.isnan(got[..., out][nan]).all())


def test_rows_outside_the_pool_and_the_table_are_left_out():
    """A page id outside the pool, a row past max_pages and a length too
    short for the tokens: nothing is written for them, the others arrive."""
    rng = np.random.default_rng(13)
    pool = Pool(rng, [20, 20, 20, 20], 0, 1, 64, 16, "f16")
    pool.table[1, 1] = pool.npages  # first row outside
    pool.table[2, 1] = -1
    pool.lens[3] = 2 * 16 + 3       # past max_pages
    k0, v0 = pool.k.clone(), pool.v.clone()
    x = torch.randn(4, 192, device="cuda").half()
    q = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    src = g.KvSource(g.ELEM_F16, 1, x.data_ptr(), x.data_ptr() + 128, x.data_ptr() + 256, 192)
    pool.kv().append(pool.batch(4), src, q.data_ptr(), 64)
    pool.lens[:] = 0                # and a sequence of no rows
    pool.kv().append(pool.batch(4), src, q.data_ptr(), 64)
    torch.cuda.synchronize()
    assert torch.equal(q, x[:, :64])
    p, o = int(pool.table_host[0, 1]), 19 % 16
    assert torch.equal(pool.k[p, 0, o], x[0, 64:128]) and torch.equal(pool.v[p, 0, o], x[0, 128:])
    k1, v1 = pool.k.clone(), pool.v.clone()
    k1[p, 0, o], v1[p, 0, o] = k0[p, 0, o], v0[p, 0, o]
    assert torch.equal(k1, k0) and torch.equal(v1, v0)


def test_queries_alone_and_keys_alone():
    rng = np.random.default_rng(15)
    pool = Pool(rng, [5, 7], 0, 2, 128, 16, "f16")
    k0, v0 = pool.k.clone(), pool.v.clone()
    x = torch.randn(2, 4, 128, device="cuda").half()
    q = torch.zeros(2, 4 * 128, dtype=torch.float16, device="cuda")
    pool.kv().append(pool.batch(2), g.KvSource(g.ELEM_F16, 4, x.data_ptr(), None, None, 512), q.data_ptr(), 512)
    torch.cuda.synchronize()
    assert torch.equal(q.view(2, 4, 128), x) and torch.equal(pool.k, k0) and torch.equal(pool.v, v0)
    pool.kv().append(pool.batch(2), g.KvSource(g.ELEM_F16, 0, None, x.data_ptr(), x.data_ptr() + 512, 512))
    torch.cuda.synchronize()
    for i, r in enumerate((4, 6)):
        p = int(pool.table_host[i, 0])
        assert torch.equal(pool.k[p, :, r], x[i, :2]) and torch.equal(pool.v[p, :, r], x[i, 2:])


def test_queries_in_place():
    rng = np.random.default_rng(17)
    pool = Pool(rng, [5] * 40, 0, 2, 256, 16, "bf16")
    x = torch.randn(40, 8, 256, device="cuda").bfloat16()
    cs = rope_table(8, 256).cuda()
    outs = []
    for dst in (torch.zeros_like(x), x):
        src = g.KvSource(g.ELEM_BF16, 4, x.data_ptr(), x.data_ptr() + 2048, x.data_ptr() + 2048 + 1024, 2048,
                         rope=cs.data_ptr(), rope_rows=8, rope_dims=256)
        pool.kv().append(pool.batch(40), src, dst.data_ptr(), 2048)
        torch.cuda.synchronize()
        outs.append(dst[:, :4].clone())
    assert torch.equal(*outs)


def test_captured_append_replays_with_the_lengths_of_the_moment():
    rng = np.random.default_rng(19)
    pool = Pool(rng, [30, 30, 30], 0, 1, 64, 16, "f16")
    x = torch.randn(3, 192, device="cuda").half()
    q = torch.zeros(3, 64, dtype=torch.float16, device="cuda")
    src = g.KvSource(g.ELEM_F16, 1, x.data_ptr(), x.data_ptr() + 128, x.data_ptr() + 256, 192)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.kv().append(pool.batch(3), src, q.data_ptr(), 64, torch.cuda.current_stream().cuda_stream)
    for n in (1, 16, 17, 30):
        pool.lens.fill_(n)
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for i in range(3):
            p, o = int(pool.table_host[i, (n - 1) // 16]), (n - 1) % 16
            assert torch.equal(pool.k[p, 0, o], x[i, 64:128]) and torch.equal(pool.v[p, 0, o], x[i, 128:])
        assert torch.equal(q, x[:, :64])
