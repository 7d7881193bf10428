"""The operators that carry an answer on, token by token, from a shared state:
keys and values appended to a paged cache (with the heads' norms and the
rotation on the way), attention of a batch whose sequences share a long
prefix, and sampling of the next token from given random numbers.

`run` computes them plainly (elementary torch operations in 32 bits, in 64
where sums decide which token is drawn) or, with `own`, calls the
framework's kernels: `PagedKv.append`, `PagedKv.attention` and `sample`.

Head counts, widths, states and batches are those of the benchmark
configurations (the 270M and 4B shapes, the per-layer-input family with
512-wide heads, the encoder's 64-wide heads; 12 and 208 questions on states
of 2,000 and 8,000 tokens) and of generic decoders around them; vocabularies
are the pruned 25,000 rows and generic full ones.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROPE_THETA, EPS = 1e6, 1e-6
LAYOUTS = {"half": 0, "interleaved": 1, "head_half": 2}


# ------------------------------------------------------------------ cases

def listed() -> list[dict]:
    return [
        # one decode step of 12 answers on the 270M shape: the smallest append, latency alone
        dict(name="append_step_270m", kind="append", nseq=12, new=1, before=40, heads=4, kv_heads=1, head_dim=256,
             page=64, src="f32", dtype="f16", layout="half", rope_dims=256, norms=True),
        # a state's tail with 208 ragged questions at the 4B shape, straight from the f32 projection
        dict(name="append_questions_4b", kind="append", nseq=208, new=40, before=17, heads=8, kv_heads=4,
             head_dim=256, page=64, src="f32", dtype="f16", layout="half", rope_dims=256, norms=True),
        # a long prompt of a generic decoder: no norms, a quarter of the interleaved head rotated, 16-row pages
        dict(name="append_prompt_bf16", kind="append", nseq=3, new=7001, before=0, heads=32, kv_heads=8,
             head_dim=128, page=16, src="bf16", dtype="bf16", layout="interleaved", rope_dims=32, norms=False),
        # 12 answers one token on, over the headline 2,000-token state
        dict(name="attend_step_270m", kind="attention", nseq=12, new=1, before=24, prefix=2000, heads=4, kv_heads=1,
             head_dim=256, page=64, dtype="f16", window=0),
        # 208 answers one token on, over an 8,000-token state
        dict(name="attend_step_4b", kind="attention", nseq=208, new=1, before=60, prefix=8000, heads=8, kv_heads=4,
             head_dim=256, page=64, dtype="f16", window=0),
        # a long conversation forked 64 ways: 65,521 shared keys and up to 2,047 of each answer's own
        dict(name="attend_step_long", kind="attention", nseq=64, new=1, before=2047, prefix=65521, heads=32,
             kv_heads=8, head_dim=128, page=16, dtype="bf16", window=0),
        # 512-wide heads: ragged questions of up to 56 tokens on a 2,000-token state
        dict(name="attend_questions_e2b", kind="attention", nseq=12, new=56, before=0, prefix=2000, heads=8,
             kv_heads=1, head_dim=512, page=32, dtype="bf16", window=0),
        # 208 questions of 40 tokens over the 8,000-token state: the largest product
        dict(name="attend_questions_4b", kind="attention", nseq=208, new=40, before=0, prefix=8000, heads=8,
             kv_heads=4, head_dim=256, page=64, dtype="f16", window=0),
        # one answer's next token from the pruned vocabulary: latency alone
        dict(name="sample_one", kind="sample", rows=1, vocab=25_000, dtype="f32", mode="chat"),
        # the 208 answers' next tokens, each with its own settings
        dict(name="sample_208_mixed", kind="sample", rows=208, vocab=25_000, dtype="f32", mode="mixed"),
        # a full vocabulary in bf16, nucleus sampling
        dict(name="sample_nucleus", kind="sample", rows=64, vocab=262_144, dtype="bf16", mode="nucleus"),
        # a large batch over an odd full vocabulary, each row with its own settings
        dict(name="sample_batch_mixed", kind="sample", rows=256, vocab=128_257, dtype="f32", mode="mixed"),
    ]


#: (heads, kv_heads, head_dim): the 270M / 1B, 4B and E2B shapes (256 and 512 wide), the encoder's heads, generic ones
SHAPES = [(4, 1, 256), (8, 4, 256), (8, 1, 256), (8, 1, 512), (12, 12, 64), (32, 8, 128), (15, 5, 64), (28, 4, 128)]
MODES = ["chat", "topk", "topp", "nucleus", "minp", "plain", "greedy", "mixed"]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "attention", "attention", "sample"])
    if kind == "sample":
        vocab = _log_int(rng, 1_000, 262_144)
        rows = _log_int(rng, 1, max(2, min(256, 32_800_000 // vocab)))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "f32", "bf16", "f16"]),
                    mode=rng.choice(MODES))
    heads, kv_heads, hd = rng.choice(SHAPES)
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "append":
        nseq = _log_int(rng, 1, 256)
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(3, 16_000_000 // (heads + kv_heads) // hd // nseq))
        new = min(new, 8192)
        layout = rng.choice(["half", "interleaved", "head_half"])
        return dict(kind=kind, nseq=nseq, new=new, before=rng.randint(0, 200), heads=heads, kv_heads=kv_heads,
                    head_dim=hd, page=page, src=rng.choice(["f32", "f32", dtype]), dtype=dtype, layout=layout,
                    rope_dims=rng.choice([hd, hd, hd // 2, hd // 4]), norms=rng.random() < 0.6)
    nseq = _log_int(rng, 1, 256)
    new = 1 if rng.random() < 0.6 else _log_int(rng, 2, max(3, min(512, 8192 // nseq)))
    before = _log_int(rng, 1, 4096) if rng.random() < 0.7 else 0
    prefix = 0 if rng.random() < 0.15 else _log_int(rng, 16, 65_536)
    # no more work than the largest listed case, and no more keys than the longest
    while 4.0 * heads * hd * nseq * new * (prefix + before + new) > 5e11 or nseq * heads * new * (prefix + before) > 5e8:
        prefix, before = prefix // 2, before // 2
    while nseq * (before + new) * kv_heads * hd > 1.2e8:
        before, nseq = before // 2, (nseq + 1) // 2
    return dict(kind=kind, nseq=nseq, new=new, before=before, prefix=prefix, heads=heads, kv_heads=kv_heads,
                head_dim=hd, page=page, dtype=dtype, window=rng.choice([0, 0, 512, 1024]))


# ---------------------------------------------------------------- prepare

def _lengths(case) -> tuple[np.ndarray, np.ndarray]:
    """(new tokens, keys before them) of each sequence: the first as given,
    the others from half of it up; single tokens stay single."""
    r = np.random.default_rng(case["nseq"] * 1009 + case["new"] * 31 + case["before"])
    n, top, old = case["nseq"], case["new"], case["before"]
    new = r.integers((top + 1) // 2, top + 1, n)
    before = r.integers(old // 2, old + 1, n)
    new[0], before[0] = top, old
    return new, before


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(DEV)


def _rope_table(rows: int, dims: int) -> torch.Tensor:
    """[rows][dims / 2] (cos, sin) pairs, angles in 64 bits."""
    f = ROPE_THETA ** (-torch.arange(0, dims, 2, dtype=torch.float64, device=DEV) / dims)
    ang = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def _prepare_cache(case, seed) -> dict:
    """A page pool holding the shared prefix and every sequence's own rows
    (pages in shuffled order, a few belonging to nobody), with its tables."""
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rng = np.random.default_rng(seed)
    new, before = _lengths(case)
    page, kv, hd = case["page"], case["kv_heads"], case["head_dim"]
    lens = new + before
    own_pages = -(-lens // page)
    pre_pages = -(-case.get("prefix", 0) // page)
    total = int(own_pages.sum() + pre_pages) + 3
    ids = rng.permutation(total)
    most = int(own_pages.max())
    table = np.zeros((case["nseq"], most), np.int64)
    at = pre_pages
    for s, n in enumerate(own_pages):
        table[s, :n] = ids[at:at + n]
        at += n
    dt = TYPES[case["dtype"]]
    shape = (total, kv, page, hd)
    st = dict(case=case, gen=gen, tokens=int(new.sum()), max_pages=most, pages=total,
              k=_randn(gen, *shape).to(dt), v=_randn(gen, *shape).to(dt), lens=_i32(lens), table=_i32(table),
              prefix_table=_i32(ids[:max(pre_pages, 1)]), prefix=case.get("prefix", 0),
              start=None if case["new"] == 1 else _i32(np.concatenate([[0], np.cumsum(new)])))
    return st


def _params(mode: str, rows: int, rng):
    """Temperature, top-k, top-p and min-p of each row (0 / 0 / 1 / 0: greedy, all, all, all)."""
    one = {"chat": (0.7, 40, 0.95, 0.0), "topk": (1.0, 200, 1.0, 0.0), "topp": (0.8, 0, 0.9, 0.0),
           "nucleus": (1.0, 0, 0.95, 0.0), "minp": (1.2, 0, 1.0, 0.05), "plain": (1.0, 0, 1.0, 0.0),
           "greedy": (0.0, 0, 1.0, 0.0), "wide": (1.5, 3000, 0.98, 0.01)}
    pick = list(one) if mode == "mixed" else [mode]
    p = np.array([one[pick[i % len(pick)]] for i in range(rows)], np.float64)
    return (torch.from_numpy(p[:, 0].astype(np.float32)).to(DEV), _i32(p[:, 1]),
            torch.from_numpy(p[:, 2].astype(np.float32)).to(DEV), torch.from_numpy(p[:, 3].astype(np.float32)).to(DEV))


def _prepare_sample(case, seed) -> dict:
    """Logits as a language model gives them: a bell of unlikely tokens and a
    few dozen likely ones per row; every seventh row keeps to a grammar that
    masks all but some hundred tokens; rows lie 8 elements wider apart than
    the vocabulary (rounded up)."""
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rows, vocab = case["rows"], case["vocab"]
    ld = (vocab + 15) // 8 * 8
    z = 2.2 * _randn(gen, rows, vocab)
    likely = torch.randint(vocab, (rows, 40), generator=gen, device=DEV)
    z.scatter_add_(1, likely, 14.0 * torch.rand(rows, 40, generator=gen, device=DEV))
    allowed = torch.rand(rows, vocab, generator=gen, device=DEV) < 100.0 / vocab
    masked = (torch.arange(rows, device=DEV) % 7 == 6)[:, None] & ~allowed
    z.masked_fill_(masked, -math.inf)
    logits = torch.zeros(rows, ld, dtype=TYPES[case["dtype"]], device=DEV)
    logits[:, :vocab] = z
    temp, top_k, top_p, min_p = _params(case["mode"], rows, np.random.default_rng(seed))
    return dict(case=case, logits=logits, ld=ld, temperature=temp, top_k=top_k, top_p=top_p, min_p=min_p,
                u=torch.rand(rows, generator=gen, device=DEV), workspace=torch.empty(0, dtype=torch.uint8, device=DEV),
                tokens=torch.zeros(rows, dtype=torch.int32, device=DEV),
                logprob=torch.zeros(rows, dtype=torch.float32, device=DEV))


def prepare(case, seed):
    if case["kind"] == "sample":
        return _prepare_sample(case, seed)
    st = _prepare_cache(case, seed)
    gen, t, H, KV, D = st["gen"], st["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        # the fused projection's rows [q heads | k heads | v heads]
        st["qkv"] = (1.5 * _randn(gen, t, (H + 2 * KV) * D)).to(TYPES[case["src"]])
        st["rope"] = _rope_table(int(st["lens"].max()) + 8, case["rope_dims"])
        if case["norms"]:
            st["q_norm"], st["k_norm"] = (1.0 + 0.3 * _randn(gen, D) for _ in range(2))
        st["q_out"] = torch.zeros(t, H, D, dtype=TYPES[case["dtype"]], device=DEV)
        return st
    # normed queries of a trained head are longer than a random key's chance product
    st["q"] = (1.7 * _randn(gen, t, H, D)).to(TYPES[case["dtype"]])
    st["out"] = torch.zeros_like(st["q"])
    st["lse"] = torch.zeros(t, H, dtype=torch.float32, device=DEV)
    st["workspace"] = torch.empty(0, dtype=torch.uint8, device=DEV)
    return st


# ------------------------------------------------------- run: plain forms

def _token_places(st):
    """(sequence, row in the sequence) of each new token."""
    case, lens = st["case"], st["lens"].long()
    t = torch.arange(st["tokens"], device=DEV)
    if st["start"] is None:
        return t, lens - 1
    start = st["start"].long()
    seq = (t[:, None] >= start[None, 1:]).sum(1)
    return seq, lens[seq] - (start[seq + 1] - t)


def _rms(x, w):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y if w is None else y * w


def _rotate(x, cs, layout):
    """x [t][heads][D] by cs [t][dims / 2][2]."""
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    n, D = cs.shape[1], x.shape[-1]
    at = torch.arange(n, device=DEV)
    a, b = {"half": (at, at + n), "interleaved": (2 * at, 2 * at + 1), "head_half": (at, at + D // 2)}[layout]
    y = x.clone()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def _plain_append(st):
    case = st["case"]
    H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
    seq, row = _token_places(st)
    x = st["qkv"].float().view(-1, H + 2 * KV, D)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    if case["norms"]:
        q, k, v = _rms(q, st["q_norm"]), _rms(k, st["k_norm"]), _rms(v, None)
    cs = st["rope"][row]
    st["q_out"].copy_(_rotate(q, cs, case["layout"]) * D ** -0.5)
    where = (st["table"].long()[seq, row // case["page"]], slice(None), row % case["page"])
    st["k"][where] = _rotate(k, cs, case["layout"]).to(st["k"].dtype)
    st["v"][where] = v.to(st["v"].dtype)
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _scores(q, k, see, scale):
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    return s.masked_fill_(~see, -math.inf)


def _plain_attention(st):
    """Scores of all queries with the prefix, and of each sequence's queries
    (padded to the longest) with its own keys; one softmax over both."""
    case = st["case"]
    H, KV, D, page, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"], st["prefix"]
    T, B, G = st["tokens"], case["nseq"], H // KV
    window = case["window"] or 1 << 30
    seq, row = _token_places(st)
    q = st["q"].float().view(T, KV, G, D).permute(1, 0, 2, 3).contiguous()  # [KV][T][G][D]
    kp, vp = (x[st["prefix_table"].long()].permute(1, 0, 2, 3).reshape(KV, -1, D)[:, :P].float()
              for x in (st["k"], st["v"]))
    key = torch.arange(P, device=DEV)
    see = (P + row)[:, None] - key[None] < window
    see = see[:, None].expand(T, G, P).reshape(1, T * G, P)
    sp = _scores(q.view(KV, T * G, D), kp, see, D ** -0.5).view(KV, T, G, P)
    # own keys: [B][KV][rows][D], the queries scattered to [B][KV][new][G]
    own_k, own_v = (x[st["table"].long()].permute(0, 2, 1, 3, 4).reshape(B, KV, -1, D).float()
                    for x in (st["k"], st["v"]))
    rows, n = own_k.shape[2], case["new"]
    slot = torch.arange(T, device=DEV) - (st["start"].long()[seq] if st["start"] is not None else seq)
    qb = torch.zeros(B, KV, n, G, D, device=DEV)
    qb[seq, :, slot] = q.permute(1, 0, 2, 3)
    at = torch.zeros(B, n, dtype=torch.long, device=DEV)
    at[seq, slot] = row
    key = torch.arange(rows, device=DEV)
    see = (key <= at[..., None]) & (at[..., None] - key < window)
    see = see[:, None, :, None].expand(B, 1, n, G, rows).reshape(B, 1, n * G, rows)
    so = _scores(qb.view(B, KV, n * G, D), own_k, see, D ** -0.5).view(B, KV, n, G, rows)
    most = torch.full((KV, T, G), -math.inf, device=DEV)
    if P:
        most = sp.amax(-1)
    mb = so.amax(-1)[seq, :, slot].permute(1, 0, 2)
    most = torch.maximum(most, mb)
    sp.sub_(most[..., None]).exp_()
    mo = torch.zeros(B, KV, n, G, device=DEV)
    mo[seq, :, slot] = most.permute(1, 0, 2)
    so.sub_(mo[..., None]).exp_()
    total = sp.sum(-1) + so.sum(-1)[seq, :, slot].permute(1, 0, 2)
    o = torch.matmul(sp.view(KV, T * G, P), vp).view(KV, T, G, D)
    oo = torch.matmul(so.view(B, KV, n * G, rows), own_v).view(B, KV, n, G, D)[seq, :, slot]
    o = (o + oo.permute(1, 0, 2, 3)) / total[..., None]
    st["out"].copy_(o.permute(1, 0, 2, 3).reshape(T, H, D))
    st["lse"].copy_((most + total.log()).permute(1, 0, 2).reshape(T, H))
    return {"out": st["out"], "lse": st["lse"]}


def _plain_sample(st):
    """The definition, in 64 bits: a tie goes to the lowest index, a token is
    kept by top-p while the mass before it is under p, and the drawn token is
    the first kept one, in vocabulary order, whose running mass exceeds u
    times the kept mass."""
    V = st["case"]["vocab"]
    z = st["logits"][:, :V].double()
    greedy = st["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(st["temperature"]), st["temperature"]).double()[:, None]
    w = ((z - z.amax(1, keepdim=True)) / t).exp()
    order = z.sort(dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = torch.where(st["top_k"] <= 0, torch.full_like(st["top_k"], V), st["top_k"]).long()[:, None]
    k = torch.where(greedy[:, None], torch.ones_like(k), k)
    place = torch.arange(V, device=DEV)[None]
    ws = ws.masked_fill_(place >= k, 0.0)
    before = ws.cumsum(1) - ws
    p = st["top_p"].double()[:, None]
    keep = (place < k) & ((before < p * ws.sum(1, keepdim=True)) | (p >= 1) | (place == 0))
    keep &= ws >= st["min_p"].double()[:, None]
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    w = w.masked_fill_(~kept, 0.0)
    run_ = w.cumsum(1)
    total = run_[:, -1:]
    tok = (run_ <= st["u"].double()[:, None] * total).sum(1, keepdim=True)
    st["tokens"].copy_(tok[:, 0])
    st["logprob"].copy_((w.gather(1, tok) / total).log()[:, 0])
    return {"tokens": st["tokens"], "logprob": st["logprob"]}


# -------------------------------------------------- run: the framework's

def _batch(g, st):
    return g.PagedBatch(st["case"]["nseq"], st["tokens"], st["lens"].data_ptr(), st["table"].data_ptr(),
                        st["max_pages"], st["start"].data_ptr() if st["start"] is not None else None,
                        st["prefix_table"].data_ptr(), st["prefix"])


def _cache(g, st):
    case = st["case"]
    return g.PagedKv(st["k"].data_ptr(), st["v"].data_ptr(), st["pages"], case["kv_heads"], case["page"],
                     case["head_dim"], {"f16": g.ELEM_F16, "bf16": g.ELEM_BF16}[case["dtype"]])


def _room(st, nbytes: int):
    """The state's workspace, made once for its sizes."""
    if st["workspace"].numel() < nbytes:
        st["workspace"] = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    return st["workspace"].data_ptr(), st["workspace"].numel()


def _own(st):
    import grande_amd as g

    case = st["case"]
    stream = torch.cuda.current_stream().cuda_stream
    elem = {"f32": g.ELEM_F32, "f16": g.ELEM_F16, "bf16": g.ELEM_BF16}
    if case["kind"] == "sample":
        ws, n = _room(st, g.sample_workspace(case["rows"], case["vocab"]))
        g.sample(st["logits"].data_ptr(), elem[case["dtype"]], case["rows"], case["vocab"], st["ld"],
                 st["u"].data_ptr(), st["tokens"].data_ptr(), st["logprob"].data_ptr(),
                 temperature=st["temperature"].data_ptr(), top_k=st["top_k"].data_ptr(), top_p=st["top_p"].data_ptr(),
                 min_p=st["min_p"].data_ptr(), workspace=ws, workspace_bytes=n, stream=stream)
        return {"tokens": st["tokens"], "logprob": st["logprob"]}
    kv, b = _cache(g, st), _batch(g, st)
    H, KV, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        x, size = st["qkv"].data_ptr(), st["qkv"].element_size()
        norms = case["norms"]
        src = g.KvSource(elem[case["src"]], H, x, x + H * D * size, x + (H + KV) * D * size, (H + 2 * KV) * D,
                         rope=st["rope"].data_ptr(), rope_rows=st["rope"].shape[0], rope_dims=case["rope_dims"],
                         rope_layout=LAYOUTS[case["layout"]], q_norm=st["q_norm"].data_ptr() if norms else None,
                         k_norm=st["k_norm"].data_ptr() if norms else None, v_norm=norms, eps=EPS, q_scale=D ** -0.5)
        kv.append(b, src, st["q_out"].data_ptr(), H * D, stream)
        return {"q": st["q_out"], "k": st["k"], "v": st["v"]}
    ws, n = _room(st, kv.attention_workspace(b, H))
    kv.attention(b, H, st["q"].data_ptr(), H * D, st["out"].data_ptr(), H * D, D ** -0.5, window=case["window"],
                 lse=st["lse"].data_ptr(), workspace=ws, workspace_bytes=n, stream=stream)
    return {"out": st["out"], "lse": st["lse"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- work

def _size(name: str) -> int:
    return 4 if name == "f32" else 2


def work(case) -> dict:
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * _size(case["dtype"]) + 28.0 * case["rows"], "flops": 3.0 * n}
    new, before = _lengths(case)
    H, KV, D, t = case["heads"], case["kv_heads"], case["head_dim"], int(new.sum())
    if case["kind"] == "append":
        rows = int((new + before).max())
        bytes_ = t * D * ((H + 2 * KV) * (_size(case["src"]) + 2.0)) + 4.0 * min(t, rows) * case["rope_dims"]
        return {"bytes": bytes_, "flops": t * D * (10.0 * H + 7 * KV)}
    P, w = case["prefix"], case["window"] or 1 << 30
    pairs, keys, first = 0, 0, P
    for n, b in zip(new.tolist(), before.tolist()):
        at = b + np.arange(n)
        pairs += int(np.minimum(at + 1, w).sum() + np.minimum(P, np.maximum(0, w - at - 1)).sum())
        keys += min(b + n, w + n - 1)
        first = min(first, max(0, P + b - w + 1))
    keys += P - first
    return {"bytes": 2.0 * D * (2 * keys * KV + 2 * t * H) + 4.0 * t * H, "flops": 4.0 * D * H * pairs}


# ------------------------------------------------------------------ exact

def _exact_append(st):
    case = st["case"]
    H, KV, D, page, n = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["rope_dims"] // 2
    new, before = _lengths(case)
    x = st["qkv"].double().reshape(-1, H + 2 * KV, D)
    if case["norms"]:
        x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt()
        x[:, :H] *= st["q_norm"].double()
        x[:, H:H + KV] *= st["k_norm"].double()
    pos = torch.from_numpy(np.concatenate([b + np.arange(k) for k, b in zip(new, before)])).to(DEV)
    z = torch.view_as_complex(st["rope"].double())[pos][:, None]
    first = {"half": slice(0, n), "interleaved": slice(0, 2 * n, 2), "head_half": slice(0, n)}[case["layout"]]
    second = {"half": slice(n, 2 * n), "interleaved": slice(1, 2 * n, 2),
              "head_half": slice(D // 2, D // 2 + n)}[case["layout"]]
    r = torch.complex(x[:, :H + KV, first].contiguous(), x[:, :H + KV, second].contiguous()) * z
    x[:, :H + KV, first], x[:, :H + KV, second] = r.real, r.imag
    k, v = st["k"].double(), st["v"].double()
    table, at = st["table"].cpu().numpy(), 0
    for s, (m, b) in enumerate(zip(new.tolist(), before.tolist())):
        rows = b + np.arange(m)
        pages, rows = torch.from_numpy(table[s, rows // page]).long().to(DEV), torch.from_numpy(rows % page).to(DEV)
        k[pages, :, rows] = x[at:at + m, H:H + KV]
        v[pages, :, rows] = x[at:at + m, H + KV:]
        at += m
    return {"q": x[:, :H] / math.sqrt(D), "k": k, "v": v}


def _exact_attention(st):
    case = st["case"]
    H, KV, D, P = case["heads"], case["kv_heads"], case["head_dim"], st["prefix"]
    new, before = _lengths(case)
    w = case["window"] or 1 << 30

    def rows(x, table, n):
        return x[table.long()].transpose(0, 1).flatten(1, 2)[:, :n].double()

    kp, vp = (rows(x, st["prefix_table"], P) for x in (st["k"], st["v"]))
    out, lse, at = [], [], 0
    for s, (n, b) in enumerate(zip(new.tolist(), before.tolist())):
        k, v = (torch.cat([a, rows(x, st["table"][s], n + b)], 1) for a, x in ((kp, st["k"]), (vp, st["v"])))
        q = st["q"][at:at + n].double().view(n, KV, H // KV, D)
        pos = P + b + torch.arange(n, device=DEV)
        back = pos[:, None] - torch.arange(P + n + b, device=DEV)
        hide = (back < 0) | (back >= w)
        o, l = [], []
        for g in range(KV):
            sc = (q[:, g].reshape(-1, D) @ k[g].T.contiguous() / math.sqrt(D)).view(n, H // KV, -1)
            sc = sc.masked_fill(hide[:, None], -math.inf)
            l.append(torch.logsumexp(sc, -1))
            o.append(((sc - l[-1][..., None]).exp().view(-1, P + n + b) @ v[g]).view(n, H // KV, D))
        out.append(torch.cat(o, 1))
        lse.append(torch.cat(l, 1))
        at += n
    return {"out": torch.cat(out), "lse": torch.cat(lse)}


def _exact_sample(st):
    """Row by row: a stable sort of the values, cumulative masses, and the
    drawn token found by bisection of the kept masses in vocabulary order."""
    V = st["case"]["vocab"]
    temp, top_k, top_p, min_p, u = (st[n].double().cpu().numpy()
                                    for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    tokens, logprob = [], []
    for r in range(st["case"]["rows"]):
        z = st["logits"][r, :V].double().cpu().numpy()
        if temp[r] <= 0:
            tokens.append(int(z.argmax()))
            logprob.append(0.0)
            continue
        w = np.exp((z - z.max()) / temp[r])
        order = np.argsort(-z.astype(np.float32), kind="stable")
        order = order[:int(top_k[r]) if 0 < top_k[r] < V else V]
        if top_p[r] < 1:
            mass = np.cumsum(w[order])
            order = order[:max(1, int(np.searchsorted(mass - w[order], top_p[r] * mass[-1], "left")))]
        order = np.sort(order[w[order] >= min_p[r]])
        mass = np.cumsum(w[order])
        i = int(np.searchsorted(mass, u[r] * mass[-1], "right"))
        tokens.append(int(order[i]))
        logprob.append(math.log(w[order[i]] / mass[-1]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device=DEV),
            "logprob": torch.tensor(logprob, dtype=torch.float64, device=DEV)}


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](st)
