"""omg_dev_sample (sample) against the definition in 64 bits, token for token:
filters alone and together, ties, masks, infinities, odd vocabularies and
strides, types, one row and many, what parameters outside their range do.

The tokens have to be equal (the masses' rounding, 2^-43 of the largest
weight a token, moves a border by less than the random numbers' spacing can
meet); the log probability is a 64-bit value rounded to f32, its mass off by
at most vocab 2^-43."""
from __future__ import annotations

import math

import numpy as np
import pytest

import grande_amd as g
from paged import ELEM, TYPES

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def plain(z, u, temp=1.0, k=0, p=1.0, mp=0.0):
    """(token, log probability) of one row, from the definition."""
    z = np.where(np.isnan(z), -np.inf, np.asarray(z, np.float64))
    if not (z > -np.inf).any():
        return -1, -math.inf
    m = z.max()
    if not temp > 0:
        return int(z.argmax()), 0.0
    with np.errstate(invalid="ignore"):
        d = np.where(z == m, 0.0, z - m)
        w = np.where(z == -np.inf, 0.0, np.where(d == 0, 1.0, np.exp(d / float(np.float32(temp)))))
    w[np.isnan(w)] = 0.0
    order = np.argsort(-(z + 0.0), kind="stable")
    order = order[z[order] > -np.inf]
    if 0 < k < len(z):
        order = order[:k]
    if p < 1:
        ws = w[order]
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        n = int((before < float(np.float32(p)) * ws.sum()).sum())
        order = order[:max(1, n)]
    if mp > 0:
        order = order[w[order] >= min(1.0, float(np.float32(mp)))]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    uu = 0.0 if not u > 0 else min(float(u), 1.0)
    at = min(int(np.searchsorted(run, uu * run[-1], "right")), len(kept) - 1)
    while w[kept[at]] == 0.0 or (at > 0 and run[at] == run[at - 1]):
        at -= 1
    return int(kept[at]), math.log(w[kept[at]] / run[-1])


def draw(z, u, temp=None, k=None, p=None, mp=None, dtype="f32", pad=0, logprob=True):
    """The framework's tokens and log probabilities; parameters per row or None."""
    rows, vocab = z.shape
    buf = torch.full((rows, vocab + pad), 1e4, dtype=TYPES[dtype], device="cuda")
    buf[:, :vocab] = torch.as_tensor(z).to(TYPES[dtype])
    ud = torch.as_tensor(np.array(u, np.float32)).cuda()
    par = {n: torch.as_tensor(np.array(v, t)).cuda() for n, v, t in
           (("temperature", temp, np.float32), ("top_k", k, np.int32), ("top_p", p, np.float32),
            ("min_p", mp, np.float32)) if v is not None}
    tok = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    lp = torch.full((rows + 1,), -7.0, device="cuda")
    ws = torch.full((g.sample_workspace(rows, vocab) + 16,), 0xFF, dtype=torch.uint8, device="cuda")
    g.sample(buf.data_ptr(), ELEM[dtype], rows, vocab, vocab + pad, ud.data_ptr(), tok.data_ptr(),
             lp.data_ptr() if logprob else None, **{n: t.data_ptr() for n, t in par.items()}, workspace=ws.data_ptr(),
             workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert int(tok[rows]) == -7 and float(lp[rows]) == -7.0
    return tok[:rows].cpu().numpy(), lp[:rows].cpu().numpy(), buf[:, :vocab].double().cpu().numpy()


def same(z, u, temp=None, k=None, p=None, mp=None, **kw):
    rows, vocab = z.shape
    full = [np.broadcast_to(np.asarray(d if v is None else v), (rows,)) for v, d in ((temp, 1.0), (k, 0), (p, 1.0), (mp, 0.0))]
    given = [None if v is None else f for v, f in zip((temp, k, p, mp), full)]
    u = np.broadcast_to(np.asarray(u, np.float32), (rows,))
    tok, lp, used = draw(z, u, *given, **kw)
    for r in range(rows):
        t, l = plain(used[r], u[r], *(f[r] for f in full))
        assert tok[r] == t, f"row {r}: token {tok[r]}, expected {t} (u {u[r]}, {[f[r] for f in full]})"
        if kw.get("logprob", True):
            assert lp[r] == l or abs(lp[r] - l) <= 2.0 ** -23 * max(1.0, abs(l)) + vocab * 2.0 ** -42, f"row {r}: {lp[r]} {l}"
    return tok


def logits(rng, rows, vocab, likely=20):
    z = 2.2 * rng.standard_normal((rows, vocab))
    for r in range(rows):
        z[r, rng.integers(0, vocab, likely)] += 14 * rng.random(likely)
    return z.astype(np.float32)


FILTERS = [dict(), dict(temp=0.7, k=40, p=0.95), dict(temp=0.7, k=40), dict(p=0.9), dict(temp=1.5, p=0.999),
           dict(temp=0.01, p=0.5), dict(mp=0.05), dict(temp=1.3, mp=0.2, p=0.8), dict(k=1), dict(k=700, p=0.97, mp=0.001),
           dict(temp=1.6, k=5000, p=0.9), dict(temp=0.0), dict(temp=30.0, p=0.7), dict(temp=30.0, k=4000),
           dict(temp=2.0, mp=1e-6), dict(temp=1.5, p=0.97, mp=1e-4), dict(temp=1.0, p=0.95)]


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 1023, 4097, 25_000, 32_769, 70_001, 262_144])
@pytest.mark.parametrize("f", range(len(FILTERS)))
def test_filters_and_vocabularies(f, vocab):
    rng = np.random.default_rng(vocab + f)
    rows = 9 if vocab < 50_000 else 4
    same(logits(rng, rows, vocab), rng.random(rows), **FILTERS[f])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("vocab,pad", [(25_000, 0), (25_001, 7), (131_072, 8), (50_257, 1)])
def test_types_and_strides(vocab, pad, dtype):
    """Half-precision logits tie by the hundred: their order is the indexes'."""
    rng = np.random.default_rng(vocab + pad)
    for f in (1, 3, 4, 6, 9, 10, 12, 13):
        same(logits(rng, 5, vocab), rng.random(5), dtype=dtype, pad=pad, **FILTERS[f])


def test_each_row_has_its_own_settings():
    rng = np.random.default_rng(5)
    z = logits(rng, 64, 9_000)
    z[6::7][:, rng.random(9_000) < 0.99] = -np.inf
    same(z, rng.random(64), temp=rng.choice([0.0, 0.5, 1.0, 2.0], 64), k=rng.choice([0, 1, 7, 50, 3000, 20_000], 64),
         p=rng.choice([1.0, 0.0, 0.3, 0.9, 0.99], 64), mp=rng.choice([0.0, 0.01, 0.5, 1.0], 64), pad=3)


@pytest.mark.parametrize("vocab", [5, 64, 1000, 40_000, 262_144])
def test_equal_logits(vocab):
    """All alike: top-k and top-p keep the first, and the token is floor(u n)."""
    z = np.zeros((6, vocab), np.float32)
    z[3] = -3.5
    u = np.array([0.0, 0.25, 0.5, 0.75, 0.99, 0.1], np.float32)
    same(z, u)
    same(z, u, k=max(1, vocab // 3))
    same(z, u, p=0.5)
    same(z, u, k=max(1, vocab // 2), p=0.25, mp=1.0)
    same(z, u, temp=0.0)


def test_zeros_of_both_signs_are_equal():
    z = np.zeros((4, 300), np.float32)
    z[:, ::2] = -0.0
    same(z, [0.0, 0.4, 0.8, 0.99], k=100)
    assert draw(z, [0.0] * 4, temp=[0.0] * 4)[0].tolist() == [0] * 4


@pytest.mark.parametrize("vocab", [200, 30_000, 100_000])
def test_masks_infinities_and_nan(vocab):
    rng = np.random.default_rng(vocab)
    z = logits(rng, 10, vocab)
    z[0] = -np.inf                                  # nothing left
    z[1] = np.nan
    z[2, 1:] = -np.inf                              # one token left
    z[3, :-1] = -np.inf
    z[4, rng.random(vocab) < 0.5] = np.nan
    z[5, [7, 90, 150]] = np.inf                     # certain tokens share the mass
    z[6] = np.finfo(np.float32).min                 # masked by the lowest value, all alike
    z[7, 10:] = np.finfo(np.float32).min
    z[8] = np.finfo(np.float32).max
    z[9, ::3] = -np.inf
    u = rng.random(10)
    for f in FILTERS:
        same(z, u, **f)
    tok, lp, _ = draw(z, u)
    assert tok[0] == tok[1] == -1 and lp[0] == lp[1] == -np.inf and tok[2] == 0 and tok[3] == vocab - 1


def test_random_numbers_at_the_ends():
    rng = np.random.default_rng(9)
    z = logits(rng, 1, 3_000).repeat(8, 0)
    z[:, :5] = -np.inf
    below = np.nextafter(np.float32(1), np.float32(0))
    u = np.array([0.0, -1.0, np.nan, below, 1.0, 5.0, -0.0, 1e-30], np.float32)
    t = same(z, u)
    assert t[0] == t[1] == t[2] == t[6] == 5 and t[4] == t[5]
    same(z, u, temp=0.8, k=50, p=0.9)


def test_parameters_outside_their_range_are_off():
    rng = np.random.default_rng(11)
    z = logits(rng, 6, 2_000)
    u = rng.random(6).astype(np.float32)
    ref = same(z, u)
    nan = np.full(6, np.nan, np.float32)
    assert np.array_equal(draw(z, u, k=np.array([-5, 0, 2000, 5000, 2 ** 31 - 1, -2 ** 31]))[0], ref)
    assert np.array_equal(draw(z, u, p=np.array([1.0, 2.0, np.inf, np.nan, 1.5, 1.0]))[0], ref)
    assert np.array_equal(draw(z, u, mp=np.array([0.0, -1.0, np.nan, -np.inf, 0.0, 0.0]))[0], ref)
    greedy = z.argmax(1)
    assert np.array_equal(draw(z, u, temp=nan)[0], greedy) and np.array_equal(draw(z, u, temp=-nan * 0 - 1)[0], greedy)
    assert np.array_equal(draw(z, u, p=np.full(6, -1.0))[0], greedy) and np.array_equal(draw(z, u, mp=np.full(6, 9.0))[0], greedy)
    same(z, u, temp=np.inf)
    same(z, u, temp=np.inf, k=17)
    same(z, u, temp=1e-30)


def test_the_draws_follow_the_distribution():
    """Evenly spaced random numbers count out every kept token's share to one."""
    rng = np.random.default_rng(13)
    z1 = logits(rng, 1, 500)
    n = 4096
    tok, lp, _ = draw(z1.repeat(n, 0), (np.arange(n) + 0.5) / n, temp=np.full(n, 0.9), k=np.full(n, 60))
    w = np.exp((z1[0].astype(np.float64) - z1.max()) / float(np.float32(0.9)))
    w[np.argsort(-z1[0], kind="stable")[60:]] = 0
    share = w / w.sum()
    assert np.abs(np.bincount(tok, minlength=500) - share * n).max() <= 1.0
    assert np.allclose(lp, np.log(share[tok]), rtol=0, atol=1e-6)


def test_without_log_probabilities_and_twice_the_same():
    rng = np.random.default_rng(15)
    z, u = logits(rng, 40, 66_000), rng.random(40)
    a = same(z, u, logprob=False, p=0.95, temp=1.4)
    for _ in range(4):
        assert np.array_equal(a, draw(z, u, p=np.full(40, 0.95), temp=np.full(40, 1.4))[0])


@pytest.mark.parametrize("vocab", [25_000, 100_000])
def test_captured_draws_replay_on_new_logits(vocab):
    rng = np.random.default_rng(17)
    z = torch.zeros(7, vocab, device="cuda")
    u, tok, lp = torch.zeros(7, device="cuda"), torch.zeros(7, dtype=torch.int32, device="cuda"), torch.zeros(7, device="cuda")
    p = torch.full((7,), 0.9, device="cuda")
    ws = torch.zeros(max(16, g.sample_workspace(7, vocab)), dtype=torch.uint8, device="cuda")

    def go():
        g.sample(z.data_ptr(), g.ELEM_F32, 7, vocab, vocab, u.data_ptr(), tok.data_ptr(), lp.data_ptr(),
                 top_p=p.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                 stream=torch.cuda.current_stream().cuda_stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(4):
        zh, uh = logits(rng, 7, vocab), rng.random(7).astype(np.float32)
        z.copy_(torch.from_numpy(zh))
        u.copy_(torch.from_numpy(uh))
        graph.replay()
        torch.cuda.synchronize()
        assert tok.tolist() == [plain(zh[r], uh[r], p=0.9)[0] for r in range(7)]
        tok.zero_()
        go()
        torch.cuda.synchronize()
        assert tok.tolist() == [plain(zh[r], uh[r], p=0.9)[0] for r in range(7)]


def test_more_rows_than_a_grids_second_size():
    """Rows past 65,535 of a long vocabulary, filters of their own: the same tokens as in a call of their own."""
    rows, vocab, tail = 66_000, 32_769, 600
    gen = torch.Generator(device="cuda").manual_seed(5)
    z = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda").normal_(0.0, 2.2, generator=gen)
    u = torch.rand(rows, device="cuda", generator=gen)
    p = torch.tensor([0.95, 0.5, 1.0], device="cuda").repeat(rows // 3)
    mp = torch.tensor([0.0, 1e-3, 0.02, 0.0], device="cuda").repeat(rows // 4)
    got = []
    for first in (0, rows - tail):
        n = rows - first
        tok = torch.full((n,), -7, dtype=torch.int32, device="cuda")
        lp = torch.zeros(n, device="cuda")
        ws = torch.empty(g.sample_workspace(n, vocab), dtype=torch.uint8, device="cuda")
        g.sample(z[first:].data_ptr(), g.ELEM_BF16, n, vocab, vocab, u[first:].data_ptr(), tok.data_ptr(), lp.data_ptr(),
                 top_p=p[first:].data_ptr(), min_p=mp[first:].data_ptr(), workspace=ws.data_ptr(),
                 workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert bool((tok >= 0).all())
        got.append((tok[-tail:].clone(), lp[-tail:].clone()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    r = rows - 2
    t, l = plain(z[r].double().cpu().numpy(), float(u[r]), 1.0, 0, float(p[r]), float(mp[r]))
    assert int(got[0][0][-2]) == t


def light_tail(rng, vocab, light, weight, mass, temp, twins=0):
    """One row: a token of weight 1, `light` tokens of `weight` each (give or take a thousandth; the first 2 `twins`
    of them side by side in pairs), and the rest, `mass` of them all together, give or take a tenth."""
    w = mass / (vocab - light - 1) * (1 + 0.1 * (2 * rng.random(vocab) - 1))
    block = rng.permutation(vocab // 64 - 1)[:light - twins + 1] * 64
    at = block + 2 * rng.integers(0, 31, len(block))
    w[at[0]] = 1.0
    w[np.concatenate([at[1:], at[1:twins + 1] + 1])] = weight * (1 + 1e-3 * (2 * rng.random(light) - 1))
    return (temp * np.log(w)).astype(np.float32)


@pytest.mark.parametrize("vocab,light,weight,mass,twins,temp,p,mp", [
    (25_000, 350, 1.2e-4, 0.08, 0, 1.0, 0.9, 5e-5),
    (25_000, 350, 1.2e-4, 0.08, 0, 1.0, 0.9, 0.0),
    (25_000, 380, 1e-4, 0.08, 0, 1.3, 0.9, 5e-5),
    (100_000, 1500, 1e-4, 0.78, 0, 1.0, 0.55, 5e-5),
    (100_000, 1500, 1e-4, 0.78, 0, 0.6, 0.55, 5e-5),
    (262_144, 4000, 2e-5, 0.23, 0, 1.0, 0.8, 1e-5),
    (100_000, 300, 1.58e-4, 0.0659, 60, 6.0, 0.9, 0.0),
    (262_144, 300, 1.58e-4, 0.0659, 60, 6.0, 0.9, 0.0)])
def test_top_p_cuts_among_light_tokens_beside_a_heavy_rest(vocab, light, weight, mass, twins, temp, p, mp):
    """The border of top_p lies among tokens lighter than (1 - p) / (2 n) of the largest, n the tokens that min_p (or
    top_p's own threshold) leaves: what top_p removes is mostly the rest of the row, not these."""
    rng = np.random.default_rng(light + vocab)
    z = np.stack([light_tail(rng, vocab, light, weight, mass, temp, twins) for _ in range(6)])
    below = np.nextafter(np.float32(1), np.float32(0))
    same(z, [0.1, 0.5, 0.97, 0.99, 0.999, below], temp=temp, p=p, mp=mp or None)
