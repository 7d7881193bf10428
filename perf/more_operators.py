"""The operators that make tokens on a long paged cache cheaper: attention for
trees of drafted tokens, moving the rows that stay (an accepted path, or what
an eviction leaves), the attention weight that each cached row gathers,
eviction of the rows that gather least, and attention over the few blocks that
a cheap score selects for each token.

`run` computes them plainly (elementary torch operations in 32 bits, in 64
where a score decides which block is taken) or, with `own`, calls the
framework's kernels: `PagedKv.attention_tree`, `keep`, `attention_weights`,
`evict`, and `block_means` with `attention_blocks`.

Head counts, widths, states and batches are those of the benchmark
configurations (the 270M and 4B shapes, the per-layer-input family with
512-wide heads, the encoder's 64-wide heads; 12 and 208 questions on states of
2,000 and 8,000 tokens) and of generic decoders around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases

def listed() -> list[dict]:
    return [
        # 12 answers' 8-token drafts on the 270M shape, over the headline state: latency alone
        dict(name="tree_step_270m", kind="tree", nseq=12, new=8, before=40, prefix=2000, heads=4, kv_heads=1,
             head_dim=256, page=64, dtype="f16", window=0),
        # 208 answers' 13-token drafts at the 4B shape over an 8,000-token state
        dict(name="tree_4b", kind="tree", nseq=208, new=13, before=60, prefix=8000, heads=8, kv_heads=4,
             head_dim=256, page=64, dtype="f16", window=0),
        # 16 long conversations, 61-token trees, small pages: the largest product
        dict(name="tree_long", kind="tree", nseq=16, new=61, before=2047, prefix=32_749, heads=32, kv_heads=8,
             head_dim=128, page=16, dtype="bf16", window=0),
        # the accepted paths of 12 drafts moved up in place: the smallest call
        dict(name="keep_path_270m", kind="keep", nseq=12, new=8, before=40, heads=4, kv_heads=1, head_dim=256,
             page=64, dtype="f16", count=5, per_head=False, apart=False),
        # lists of each KV head's own, 1,000 of 2,047 rows of 64 sequences to other pages
        dict(name="keep_rows_apart", kind="keep", nseq=64, new=1, before=2046, heads=32, kv_heads=8, head_dim=128,
             page=16, dtype="bf16", count=1000, per_head=True, apart=True),
        # 12 answers one token on, the weight of their 2,000 rows each
        dict(name="weights_step_270m", kind="weights", nseq=12, new=1, before=2000, heads=4, kv_heads=1, head_dim=256,
             page=64, dtype="f16", window=0),
        # 64 long sequences one token on
        dict(name="weights_step_long", kind="weights", nseq=64, new=1, before=8190, heads=32, kv_heads=8,
             head_dim=128, page=16, dtype="bf16", window=0),
        # a whole 8,000-token prompt at the 4B shape
        dict(name="weights_prompt_4b", kind="weights", nseq=1, new=8000, before=0, heads=8, kv_heads=4, head_dim=256,
             page=64, dtype="f16", window=0),
        # 12 answers cut from 2,300 rows to 1,024, to other pages
        dict(name="evict_270m", kind="evict", nseq=12, new=1, before=2299, heads=4, kv_heads=1, head_dim=256, page=64,
             dtype="f16", keep=1024, recent=256),
        # 64 long sequences halved
        dict(name="evict_long", kind="evict", nseq=64, new=1, before=8190, heads=32, kv_heads=8, head_dim=128, page=16,
             dtype="bf16", keep=4095, recent=512),
        # 12 answers one token on, 32 of the 125 blocks of an 8,000-token state at the 4B shape
        dict(name="blocks_step_4b", kind="blocks", nseq=12, new=1, before=60, prefix=8000, heads=8, kv_heads=4,
             head_dim=256, page=64, dtype="f16", blocks=32),
        # a conversation forked 64 ways: 64 blocks out of some 1,040
        dict(name="blocks_step_long", kind="blocks", nseq=64, new=1, before=2047, prefix=65_521, heads=32, kv_heads=8,
             head_dim=128, page=64, dtype="bf16", blocks=64),
    ]


#: (heads, kv_heads, head_dim): the 270M / 1B, 4B and E2B shapes (256 and 512 wide), the encoder's heads, generic ones
SHAPES = [(4, 1, 256), (8, 4, 256), (8, 1, 256), (8, 1, 512), (12, 12, 64), (32, 8, 128), (15, 5, 64), (28, 4, 128)]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["tree", "keep", "weights", "weights", "evict", "blocks"])
    heads, kv_heads, hd = rng.choice(SHAPES)
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, head_dim=hd, page=rng.choice([16, 32, 64, 128]),
                dtype=rng.choice(["f16", "bf16"]))
    row = kv_heads * hd
    if kind == "tree":
        nseq, new = _log_int(rng, 1, 208), _log_int(rng, 2, 90)
        before, prefix = _log_int(rng, 1, 2048), 0 if rng.random() < 0.2 else _log_int(rng, 16, 32_768)
        # no more work than the largest listed case, and no more scores
        while 4.0 * heads * hd * nseq * new * (prefix + before + new) > 5e11 or nseq * heads * new * (prefix + before) > 1e9:
            nseq, prefix = (nseq + 1) // 2, prefix // 2
        while nseq * (before + new) * row > 6e7:
            before, nseq = before // 2, (nseq + 1) // 2
        return dict(case, nseq=nseq, new=new, before=before, prefix=prefix, window=rng.choice([0, 0, 512, 1024]))
    nseq = _log_int(rng, 1, 128)
    if kind == "keep":
        if rng.random() < 0.5:  # a path
            return dict(case, nseq=nseq, new=_log_int(rng, 2, 64), before=rng.randint(0, 200),
                        count=rng.randint(1, 16), per_head=False, apart=False)
        before = _log_int(rng, 64, max(65, min(8192, int(1.2e8) // row // nseq)))
        return dict(case, nseq=nseq, new=1, before=before, count=rng.randint(1, before), per_head=bool(rng.random() < 0.7),
                    apart=bool(rng.random() < 0.5))
    if kind == "weights":
        window = rng.choice([0, 0, 512])
        if rng.random() < 0.5:
            return dict(case, nseq=nseq, new=1, before=_log_int(rng, 16, max(17, min(16_384, int(2.6e8) // row // nseq))),
                        window=window)
        new = _log_int(rng, 2, 4096)
        before = rng.choice([0, 0, rng.randint(1, 2000)])
        while nseq * new * (new + before) * heads * hd > 6e10 or nseq * new * (new + before) * heads > 3e8:
            nseq, new = (nseq + 1) // 2, (2 * new + 2) // 3
        return dict(case, nseq=nseq, new=new, before=before, window=window)
    if kind == "evict":
        before = _log_int(rng, 64, max(65, min(16_384, int(2.6e8) // row // nseq)))
        keep = rng.randint(8, before)
        return dict(case, nseq=nseq, new=1, before=before, keep=keep, recent=rng.randint(0, keep))
    nseq, new = min(nseq, 64), rng.choice([1, 1, 1, 3])
    before, prefix = _log_int(rng, 1, 2048), 0 if rng.random() < 0.2 else _log_int(rng, 256, 65_536)
    blocks = _log_int(rng, 2, 96)
    while nseq * new * blocks * case["page"] * row > 2.7e8:
        nseq, blocks = (nseq + 1) // 2, blocks // 2 + 1
    while nseq * (before + new) * row > 1.3e8:
        before = before // 2
    return dict(case, nseq=nseq, new=new, before=before, prefix=prefix, blocks=blocks)


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


def _masks(rng, new) -> tuple[np.ndarray, np.ndarray]:
    """Random draft trees: each token a child of one of the few before it (or
    of the sequence's end).  The bits of the tokens each one sees (its
    ancestors and itself) and its depth."""
    words = (int(new.max()) + 31) // 32
    bits = np.zeros((int(new.sum()), words), np.uint32)
    depth = np.zeros(int(new.sum()), np.int64)
    at = 0
    for n in new.tolist():
        for i in range(n):
            parent = int(rng.integers(max(-1, i // 2 - 3), i))
            if parent >= 0:
                bits[at + i] = bits[at + parent]
                depth[at + i] = depth[at + parent] + 1
            bits[at + i, i // 32] |= np.uint32(1 << (i % 32))
        at += n
    return bits.view(np.int32), depth


def _lists(case, rng, new, before) -> np.ndarray:
    """The rows that stay, ascending: a path through each draft, or `count`
    random rows of each list (fewer where a sequence has fewer; -1 ends)."""
    heads = case["kv_heads"] if case["per_head"] else 1
    rows = np.full((case["nseq"], heads, case["count"]), -1, np.int64)
    for s, (n, b) in enumerate(zip(new.tolist(), before.tolist())):
        for h in range(heads):
            if case["new"] > 1:
                m = int(rng.integers(1, min(n, case["count"]) + 1))
                rows[s, h, :m] = b + np.sort(rng.permutation(n)[:m])
            else:
                m = min(n + b, case["count"])
                rows[s, h, :m] = np.sort(rng.permutation(n + b)[:m])
    return rows if case["per_head"] else rows[:, 0]


def prepare(case, seed) -> dict:
    """A page pool holding the shared prefix and every sequence's own rows
    (pages in shuffled order, a few belonging to nobody), with its tables."""
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    rng = np.random.default_rng(seed)
    kind, page, H, KV, D = case["kind"], case["page"], case["heads"], case["kv_heads"], case["head_dim"]
    new, before = _lengths(case)
    lens, B, T, P = new + before, case["nseq"], int(new.sum()), case.get("prefix", 0)
    apart = kind == "evict" or case.get("apart", False)
    to = -(-np.minimum(lens, case.get("keep", case.get("count", 0))) // page) if apart else np.zeros(B, np.int64)
    own_pages, pre_pages = -(-lens // page), -(-P // page)
    total = int(own_pages.sum() + pre_pages + to.sum()) + 3
    ids = rng.permutation(total)

    def deal(counts, at):
        t = np.zeros((B, max(1, int(counts.max()))), np.int64)
        for s, n in enumerate(counts.tolist()):
            t[s, :n] = ids[at:at + n]
            at += n
        return t, at
    table, at = deal(own_pages, pre_pages)
    to_table, _ = deal(to, at)
    dt, shape = TYPES[case["dtype"]], (total, KV, page, D)
    st = dict(case=case, tokens=T, max_pages=table.shape[1], pages=total, lens=_i32(lens), table=_i32(table), prefix=P,
              prefix_table=_i32(ids[:max(pre_pages, 1)]), k=_randn(gen, *shape).to(dt), v=_randn(gen, *shape).to(dt),
              start=None if case["new"] == 1 else _i32(np.concatenate([[0], np.cumsum(new)])),
              workspace=torch.empty(0, dtype=torch.uint8, device=DEV))
    if apart:
        st["to_table"] = _i32(to_table)
    if kind in ("tree", "weights", "blocks"):
        # normed queries of a trained head are longer than a random key's chance product
        st["q"] = (1.7 * _randn(gen, T, H, D)).to(dt)
        st["lse"] = torch.zeros(T, H, device=DEV)
        st["out"] = torch.zeros_like(st["q"])
    if kind == "tree":
        bits, depth = _masks(rng, new)
        st["mask"] = _i32(bits)
        st["positions"] = _i32(P + np.repeat(before, new) + depth)
    elif kind == "keep":
        st["rows"] = _i32(_lists(case, rng, new, before))
        st["first"] = _i32(before) if case["new"] > 1 else None
    elif kind == "weights":
        # what the step's attention left: the log sums, and the weights of the steps before
        sc, _ = _own_scores(st, lambda x: x.float())
        st["lse"].copy_(_to_tokens(st, torch.logsumexp(sc, -1)))
        st["weights"] = torch.exp(0.5 * _randn(gen, B, KV, st["max_pages"] * page))
    elif kind == "evict":
        # a few rows gather most of the weight, some have gathered none yet
        w = torch.exp(1.5 * _randn(gen, B, KV, st["max_pages"] * page))
        st["weights"] = w * (torch.rand(w.shape, generator=gen, device=DEV) > 0.05)
        st["rows"] = torch.zeros(B, KV, case["keep"], dtype=torch.int32, device=DEV)
        st["kept_weights"] = torch.zeros(B, KV, case["keep"], device=DEV)
    elif kind == "blocks":
        # neighbouring keys are alike; the means of all rows before the new ones
        st["k"].copy_(st["k"].float() + 0.5 * _randn(gen, total, KV, 1, D))
        full = np.full(total, page)
        for s, n in enumerate(before.tolist()):
            if n % page:
                full[table[s, n // page]] = n % page
        if P % page:
            full[ids[pre_pages - 1]] = P % page
        use = torch.arange(page, device=DEV) < _i32(full)[:, None]
        st["means"] = ((st["k"] * use[:, None, :, None]).sum(2, dtype=torch.float32) / _i32(full)[:, None, None])
        st["chosen"] = torch.zeros(T, KV, case["blocks"], dtype=torch.int32, device=DEV)
    return st


# ------------------------------------------------------- run: plain forms

def _token_places(st):
    """(sequence, row in the sequence, place among its new tokens) of each new token."""
    lens = st["lens"].long()
    t = torch.arange(st["tokens"], device=DEV)
    if st["start"] is None:
        return t, lens - 1, torch.zeros_like(t)
    start = st["start"].long()
    seq = (t[:, None] >= start[None, 1:]).sum(1)
    return seq, lens[seq] - (start[seq + 1] - t), t - start[seq]


def _own_rows(st, name, to):
    """Every sequence's own rows, padded to the table's width: [nseq][kv_heads][rows][head_dim]."""
    x = st[name][st["table"].long()].permute(0, 2, 1, 3, 4)
    return to(x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1]))


def _to_tokens(st, x):
    """[nseq][kv_heads][new][group] -> [tokens][heads]."""
    seq, _, slot = _token_places(st)
    return x[seq, :, slot].reshape(st["tokens"], -1)


def _own_scores(st, to):
    """Scores [nseq][kv_heads][new][group][rows] of every sequence's queries
    (padded to the longest) with its own rows, -inf where it does not see."""
    case = st["case"]
    H, KV, D, B, n = case["heads"], case["kv_heads"], case["head_dim"], case["nseq"], case["new"]
    G, seq, row, slot = H // KV, *_token_places(st)
    k = _own_rows(st, "k", to)
    rows = k.shape[2]
    qb = torch.zeros(B, KV, n, G, D, device=DEV, dtype=k.dtype)
    qb[seq, :, slot] = to(st["q"]).view(-1, KV, G, D)
    key = torch.arange(rows, device=DEV)
    see = torch.zeros(B, n, rows, dtype=torch.bool, device=DEV)
    if case["kind"] == "tree":
        w = case["window"] or 1 << 30
        base = (row - slot)[:, None]
        j = (key[None] - base).clamp(0, 32 * st["mask"].shape[1] - 1)
        bit = (st["mask"].long().gather(1, j // 32) >> (j % 32)) & 1 != 0
        near = st["positions"].long()[:, None] - (st["prefix"] + key[None]) < w
        see[seq, slot] = torch.where(key[None] < base, near, bit & (key[None] < st["lens"].long()[seq][:, None]))
    else:
        w = case["window"] or 1 << 30
        see[seq, slot] = (key[None] <= row[:, None]) & (row[:, None] - key[None] < w)
    sc = torch.matmul(qb.view(B, KV, n * G, D), k.transpose(-1, -2).contiguous()) * D ** -0.5
    sc = sc.view(B, KV, n, G, rows).masked_fill_(~see[:, None, :, None], -math.inf)
    return sc, see


def _plain_tree(st):
    """Scores of all queries with the prefix, and of each sequence's queries
    with its own rows; one softmax over both."""
    case = st["case"]
    H, KV, D, P, T, B, n = (case["heads"], case["kv_heads"], case["head_dim"], st["prefix"], st["tokens"],
                            case["nseq"], case["new"])
    G, seq, row, slot = H // KV, *_token_places(st)
    so, _ = _own_scores(st, lambda x: x.float())
    rows = so.shape[-1]
    most = so.amax(-1)[seq, :, slot].permute(1, 0, 2)  # [KV][T][G]
    q = st["q"].float().view(T, KV, G, D).permute(1, 0, 2, 3).contiguous()
    kp, vp = (x[st["prefix_table"].long()].permute(1, 0, 2, 3).reshape(KV, -1, D)[:, :P].float()
              for x in (st["k"], st["v"]))
    sp = torch.matmul(q.view(KV, T * G, D), kp.transpose(-1, -2).contiguous()).mul_(D ** -0.5).view(KV, T, G, P)
    if case["window"]:
        far = st["positions"].long()[:, None] - torch.arange(P, device=DEV) >= case["window"]
        sp.masked_fill_(far[:, None], -math.inf)
    if P:
        most = torch.maximum(most, sp.amax(-1))
    sp.sub_(most[..., None]).exp_()
    mo = torch.zeros(B, KV, n, G, device=DEV)
    mo[seq, :, slot] = most.permute(1, 0, 2)
    so.sub_(mo[..., None]).exp_()
    total = sp.sum(-1) + so.sum(-1)[seq, :, slot].permute(1, 0, 2)
    o = torch.matmul(sp.view(KV, T * G, P), vp).view(KV, T, G, D)
    v = _own_rows(st, "v", lambda x: x.float())
    oo = torch.matmul(so.view(B, KV, n * G, rows), v).view(B, KV, n, G, D)[seq, :, slot]
    o = (o + oo.permute(1, 0, 2, 3)) / total[..., None]
    st["out"].copy_(o.permute(1, 0, 2, 3).reshape(T, H, D))
    st["lse"].copy_((most + total.log()).permute(1, 0, 2).reshape(T, H))
    return {"out": st["out"], "lse": st["lse"]}


def _move(st, rows, first, to_table):
    """Row first + j of every list becomes its row rows[j]."""
    page, KV = st["case"]["page"], st["case"]["kv_heads"]
    rows = rows.long().expand(-1, KV, -1)
    s, h, j = torch.nonzero(rows >= 0, as_tuple=True)
    src = rows[s, h, j]
    dst = j if first is None else first.long()[s] + j
    fp, tp = st["table"].long()[s, src // page], to_table.long()[s, dst // page]
    for_k, for_v = st["k"][fp, h, src % page], st["v"][fp, h, src % page]
    st["k"][tp, h, dst % page] = for_k
    st["v"][tp, h, dst % page] = for_v


def _plain_keep(st):
    rows = st["rows"] if st["case"]["per_head"] else st["rows"][:, None]
    _move(st, rows, st["first"], st["to_table"] if st["case"]["apart"] else st["table"])
    return {"k": st["k"], "v": st["v"]}


def _plain_weights(st):
    """Each row's probabilities, summed over the queries that see it."""
    sc, see = _own_scores(st, lambda x: x.float())
    seq, _, slot = _token_places(st)
    lse = torch.full(sc.shape[:4], math.inf, device=DEV)
    lse[seq, :, slot] = st["lse"].view(st["tokens"], sc.shape[1], sc.shape[3])
    st["weights"] += sc.sub_(lse[..., None]).exp_().sum((2, 3))
    return {"weights": st["weights"]}


def _plain_evict(st):
    """The last `recent` rows and the heaviest of the others (ties: the first ones), in order."""
    case, lens = st["case"], st["lens"].long()[:, None, None]
    keep, w = case["keep"], st["weights"]
    at = torch.arange(w.shape[-1], device=DEV)
    rank = w.masked_fill(at >= lens, -math.inf).masked_fill((at < lens) & (at >= lens - case["recent"]), math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    if order.shape[-1] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=w.shape[-1])
    order = torch.where(order < lens, order, w.shape[-1]).sort(-1).values
    there = order < lens
    rows = torch.where(there, order, -1)
    st["rows"].copy_(rows)
    kept = w.gather(-1, rows.clamp(min=0))
    st["kept_weights"].copy_(torch.where(there, kept, 0.0))
    _move(st, rows, None, st["to_table"])
    return {"rows": st["rows"], "weights": st["kept_weights"], "k": st["k"], "v": st["v"]}


def _plain_blocks(st):
    """The means of the pages that the new rows are on; every block's score
    (the group's queries with its mean, in 64 bits); the token's own block and
    the best others; attention over their rows."""
    case = st["case"]
    page, H, KV, D, P, T, kb = (case["page"], case["heads"], case["kv_heads"], case["head_dim"], st["prefix"],
                                st["tokens"], case["blocks"])
    G, seq, row, _ = H // KV, *_token_places(st)
    table, lens = st["table"].long(), st["lens"].long()
    # (several new rows of one page take the same mean)
    touched = table[seq, row // page]
    use = (row // page * page)[:, None] + torch.arange(page, device=DEV) < lens[seq][:, None]
    mean = (st["k"][touched].double() * use[:, None, :, None]).sum(2) / use.sum(1)[:, None, None]
    st["means"][touched] = mean.float()
    np_ = -(-P // page)
    ids = torch.cat([st["prefix_table"].long()[:np_].expand(T, -1), table[seq]], 1)  # [T][blocks]
    nb = ids.shape[1]
    own_block = np_ + row // page
    qs = st["q"].double().view(T, KV, G, D).sum(2)
    if np_:
        sp = torch.matmul(qs.transpose(0, 1), st["means"][st["prefix_table"].long()[:np_]].double().permute(1, 2, 0).contiguous())
    else:
        sp = torch.zeros(KV, T, 0, dtype=torch.float64, device=DEV)
    so = torch.matmul(qs[:, :, None], st["means"][table[seq]].double().permute(0, 2, 3, 1).contiguous())[:, :, 0]
    score = torch.cat([sp.transpose(0, 1), so], 2).float()  # [T][KV][blocks]
    at = torch.arange(nb, device=DEV)
    score.masked_fill_((at > own_block[:, None])[:, None], -math.inf)
    score.masked_fill_((at == own_block[:, None])[:, None], math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :kb]
    if order.shape[-1] < kb:
        order = torch.nn.functional.pad(order, (0, kb - order.shape[-1]), value=nb)
    order = torch.where(order <= own_block[:, None, None], order, nb).sort(-1).values
    there = order <= own_block[:, None, None]
    st["chosen"].copy_(torch.where(there, order, -1))
    pick = order.clamp(max=nb - 1)
    pages = ids[torch.arange(T, device=DEV)[:, None, None], pick]
    # the rows of each block that there are
    end = torch.where(pick < np_, P - pick * page, row[:, None, None] + 1 - (pick - np_) * page)
    see = (torch.arange(page, device=DEV) < end[..., None]) & there[..., None]
    head = torch.arange(KV, device=DEV)[None, :, None]
    k = st["k"][pages, head].float().view(T, KV, kb * page, D)
    sc = torch.matmul(st["q"].float().view(T, KV, G, D), k.transpose(-1, -2).contiguous()) * D ** -0.5
    sc.masked_fill_(~see.view(T, KV, 1, kb * page), -math.inf)
    lse = torch.logsumexp(sc, -1)
    v = st["v"][pages, head].float().view(T, KV, kb * page, D)
    st["out"].copy_(torch.matmul((sc - lse[..., None]).exp_(), v).view(T, H, D))
    st["lse"].copy_(lse.view(T, H))
    return {"chosen": st["chosen"], "out": st["out"], "lse": st["lse"], "means": st["means"]}


# -------------------------------------------------- run: the framework's

def _room(st, nbytes: int):
    """The state's workspace, made once for its sizes."""
    if st["workspace"].numel() < nbytes:
        st["workspace"] = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    return dict(workspace=st["workspace"].data_ptr(), workspace_bytes=st["workspace"].numel())


def _own(st):
    import grande_amd as g

    case = st["case"]
    kind, H, KV, D = case["kind"], case["heads"], case["kv_heads"], case["head_dim"]
    stream = torch.cuda.current_stream().cuda_stream
    kv = g.PagedKv(st["k"].data_ptr(), st["v"].data_ptr(), st["pages"], KV, case["page"], D,
                   {"f16": g.ELEM_F16, "bf16": g.ELEM_BF16}[case["dtype"]])
    b = g.PagedBatch(case["nseq"], st["tokens"], st["lens"].data_ptr(), st["table"].data_ptr(), st["max_pages"],
                     st["start"].data_ptr() if st["start"] is not None else None, st["prefix_table"].data_ptr(),
                     st["prefix"])
    if kind == "tree":
        kv.attention_tree(b, H, st["q"].data_ptr(), H * D, st["out"].data_ptr(), H * D, D ** -0.5, st["mask"].data_ptr(),
                          st["mask"].shape[1], window=case["window"], positions=st["positions"].data_ptr(),
                          lse=st["lse"].data_ptr(), **_room(st, kv.attention_tree_workspace(b, H)), stream=stream)
        return {"out": st["out"], "lse": st["lse"]}
    if kind == "keep":
        to = dict(to_table=st["to_table"].data_ptr(), to_ld=st["to_table"].shape[1]) if case["apart"] else {}
        kv.keep(b, st["rows"].data_ptr(), case["count"], case["count"], per_head=case["per_head"],
                first=st["first"].data_ptr() if st["first"] is not None else None, **to, stream=stream)
        return {"k": st["k"], "v": st["v"]}
    if kind == "weights":
        kv.attention_weights(b, H, st["q"].data_ptr(), H * D, st["lse"].data_ptr(), D ** -0.5, st["weights"].data_ptr(),
                             st["weights"].shape[2], window=case["window"],
                             **_room(st, kv.attention_weights_workspace(b, H)), stream=stream)
        return {"weights": st["weights"]}
    if kind == "evict":
        kv.evict(b, case["keep"], case["recent"], st["weights"].data_ptr(), st["weights"].shape[2], st["rows"].data_ptr(),
                 kept_weights=st["kept_weights"].data_ptr(), kept_ld=case["keep"], to_table=st["to_table"].data_ptr(),
                 to_ld=st["to_table"].shape[1], stream=stream)
        return {"rows": st["rows"], "weights": st["kept_weights"], "k": st["k"], "v": st["v"]}
    kv.block_means(b, st["means"].data_ptr(), stream=stream)
    kv.attention_blocks(b, H, st["q"].data_ptr(), H * D, st["out"].data_ptr(), H * D, D ** -0.5, st["means"].data_ptr(),
                        case["blocks"], lse=st["lse"].data_ptr(), chosen=st["chosen"].data_ptr(),
                        **_room(st, kv.attention_blocks_workspace(b, H, case["blocks"])), stream=stream)
    return {"chosen": st["chosen"], "out": st["out"], "lse": st["lse"], "means": st["means"]}


def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "keep": _plain_keep, "weights": _plain_weights, "evict": _plain_evict,
            "blocks": _plain_blocks}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- work

def work(case) -> dict:
    new, before = _lengths(case)
    kind, H, KV, D, t, page = (case["kind"], case["heads"], case["kv_heads"], case["head_dim"], int(new.sum()),
                               case["page"])
    lens = new + before
    if kind == "keep":
        lists = case["nseq"] * (KV if case["per_head"] else 1)
        n = int(np.minimum(lens if case["new"] == 1 else (new + 1) // 2, case["count"]).sum())
        return {"bytes": 8.0 * n * KV * D + 4.0 * lists * case["count"], "flops": 0.0}
    if kind == "evict":
        kept = int(np.minimum(lens, case["keep"]).sum())
        return {"bytes": KV * (8.0 * kept * D + 4.0 * int(lens.sum()) + 8.0 * kept), "flops": 1.0 * KV * int(lens.sum())}
    P, w = case.get("prefix", 0), case.get("window", 0) or 1 << 30
    if kind == "blocks":
        np_, k = -(-P // page), case["blocks"]
        mine = (lens - 1) // page + 1
        take = np.minimum(np_ + mine, k)
        # the prefix's different blocks that so many chance choices hit, and the sequences' own
        share = (take - 1) / np.maximum(1, np_ + mine - 1)
        blocks = np_ * (1 - float(np.prod((1 - share) ** new))) + float((1 + (mine - 1) * share).sum())
        return {"bytes": 4.0 * D * KV * (blocks * page + np_ + int(mine.sum())) + 4.0 * t * H * D,
                "flops": 4.0 * D * H * float((new * take).sum() * page)}
    pairs, keys, first = 0, 0, P
    for n, b in zip(new.tolist(), before.tolist()):
        at = b + np.arange(n)
        if kind == "tree":
            pairs += int((np.minimum(b, w) + (at - b) // 2 + 1).sum() + np.minimum(P, np.maximum(0, w - at - 1)).sum())
        else:
            pairs += int(np.minimum(at + 1, w).sum())
        keys += min(b + n, w + n - 1)
        first = min(first, max(0, P + b - w + 1))
    if kind == "weights":
        return {"bytes": 2.0 * D * (keys * KV + t * H) + 4.0 * t * H + 8.0 * keys * KV, "flops": 2.0 * D * H * pairs}
    keys += P - first
    return {"bytes": 2.0 * D * (2 * keys * KV + 2 * t * H) + 4.0 * t * H, "flops": 4.0 * D * H * pairs}


# ------------------------------------------------------------------ exact

def _rows_of(x, table, n):
    return x[table.long()].transpose(0, 1).flatten(1, 2)[:, :n].double()


def _exact_attention(st):
    """Sequence by sequence: the outputs and log sums of a tree, or the weights of the rows."""
    case = st["case"]
    H, KV, D, P = case["heads"], case["kv_heads"], case["head_dim"], st["prefix"]
    new, before = _lengths(case)
    w, tree, at = case["window"] or 1 << 30, case["kind"] == "tree", 0
    if not tree:
        got = st["weights"].double()
    kp, vp = (_rows_of(x, st["prefix_table"], P) for x in (st["k"], st["v"]))
    out, lse = [], []
    for s, (n, b) in enumerate(zip(new.tolist(), before.tolist())):
        q = st["q"][at:at + n].double().view(n, KV, H // KV, D)
        k = torch.cat([kp, _rows_of(st["k"], st["table"][s], n + b)], 1)
        if tree:
            bits = np.unpackbits(st["mask"][at:at + n].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :n]
            hide = st["positions"][at:at + n].long()[:, None] - torch.arange(P + b, device=DEV) >= w
            hide = torch.cat([hide, torch.from_numpy(bits == 0).to(DEV)], 1)
            v = torch.cat([vp, _rows_of(st["v"], st["table"][s], n + b)], 1)
        else:
            back = b + torch.arange(n, device=DEV)[:, None] - torch.arange(n + b, device=DEV)
            hide = (back < 0) | (back >= w)
        o, l = [], []
        for g in range(KV):
            group = 0.0
            for h in range(H // KV):
                sc = (q[:, g, h] @ k[g].T.contiguous() / math.sqrt(D)).masked_fill(hide, -math.inf)
                if tree:
                    l.append(torch.logsumexp(sc, -1))
                    o.append((sc - l[-1][:, None]).exp() @ v[g])
                else:
                    group = group + (sc - st["lse"][at:at + n, g * (H // KV) + h].double()[:, None]).exp().sum(0)
            if not tree:
                got[s, g, :n + b] += group
        if tree:
            out.append(torch.stack(o, 1))
            lse.append(torch.stack(l, 1))
        at += n
    return {"out": torch.cat(out), "lse": torch.cat(lse)} if tree else {"weights": got}


def _exact_move(st, k, v, lists, first, to):
    """Copies of the cache with every list's rows where they go; a list for all heads or one for each."""
    case, page = st["case"], st["case"]["page"]
    table, to, old_k, old_v = st["table"].cpu().numpy(), to.cpu().numpy(), st["k"], st["v"]
    for s, per in enumerate(lists):
        for g in range(case["kv_heads"]):
            rows = per[g % len(per)]
            rows = rows[rows >= 0]
            dst = (int(first[s]) if first is not None else 0) + np.arange(len(rows))
            a, b, c, d = (torch.from_numpy(np.asarray(x, np.int64)).to(DEV)
                          for x in (table[s, rows // page], rows % page, to[s, dst // page], dst % page))
            k[c, g, d], v[c, g, d] = old_k[a, g, b].to(k.dtype), old_v[a, g, b].to(v.dtype)


def _exact_keep(st):
    lists = st["rows"].cpu().numpy().reshape(st["case"]["nseq"], -1, st["case"]["count"])
    k, v = st["k"].clone(), st["v"].clone()
    _exact_move(st, k, v, lists, st["first"].cpu().numpy() if st["first"] is not None else None,
                st["to_table"] if st["case"]["apart"] else st["table"])
    return {"k": k, "v": v}


def _exact_evict(st):
    case = st["case"]
    weights, lens, keep = st["weights"].cpu().numpy(), st["lens"].cpu().numpy(), case["keep"]
    rows = np.full((case["nseq"], case["kv_heads"], keep), -1, np.int64)
    kept = np.zeros(rows.shape, np.float64)
    for s in range(case["nseq"]):
        n = int(lens[s])
        for g in range(case["kv_heads"]):
            old = max(0, n - case["recent"])
            w = weights[s, g, :old]
            take = np.lexsort((np.arange(old), -w))[:max(0, keep - (n - old))]
            r = np.concatenate([np.sort(take), np.arange(old, n)])
            rows[s, g, :len(r)], kept[s, g, :len(r)] = r, weights[s, g, r]
    k, v = st["k"].clone(), st["v"].clone()
    _exact_move(st, k, v, rows, None, st["to_table"])
    return {"rows": torch.from_numpy(rows.astype(np.int32)).to(DEV), "weights": torch.from_numpy(kept).to(DEV), "k": k,
            "v": v}


def _exact_blocks(st):
    case = st["case"]
    page, H, KV, D, P, kb = (case["page"], case["heads"], case["kv_heads"], case["head_dim"], st["prefix"],
                             case["blocks"])
    new, before = _lengths(case)
    means, np_, table, pre = st["means"].double(), -(-P // page), st["table"].cpu().numpy(), st["prefix_table"].cpu().numpy()
    chosen = np.full((st["tokens"], KV, kb), -1, np.int32)
    out, lse = torch.zeros(st["tokens"], H, D, dtype=torch.float64, device=DEV), torch.zeros(st["tokens"], H, dtype=torch.float64, device=DEV)
    for s, (n, b) in enumerate(zip(new.tolist(), before.tolist())):
        for j in range(b // page, (b + n - 1) // page + 1):
            means[table[s, j]] = st["k"][table[s, j]][:, :n + b - j * page].double().mean(1).float().double()
    at = 0
    for s, (n, b) in enumerate(zip(new.tolist(), before.tolist())):
        for i in range(n):
            last = np_ + (b + i) // page
            ids = np.concatenate([pre[:np_], table[s, :last - np_ + 1]]).astype(np.int64)
            dev_ids = torch.from_numpy(ids).to(DEV)
            q = st["q"][at].double().view(KV, H // KV, D)
            score = (means[dev_ids] * q.sum(1)).sum(-1).float().cpu().numpy()  # [blocks][KV]
            ends = np.where(np.arange(last + 1) < np_, np.minimum(page, P - np.arange(last + 1) * page), page)
            ends[last] = (b + i) % page + 1
            for g in range(KV):
                take = np.sort(np.append(np.lexsort((np.arange(last), -score[:last, g]))[:kb - 1], last))
                chosen[at, g, :len(take)] = take
                pick = torch.from_numpy(take).to(DEV)
                see = torch.arange(page, device=DEV) < torch.from_numpy(ends[take]).to(DEV)[:, None]
                k, v = (x[dev_ids[pick], g].double()[see] for x in (st["k"], st["v"]))
                sc = (q[g][:, None] * k).sum(-1) / math.sqrt(D)
                l = torch.logsumexp(sc, -1)
                lse[at].view(KV, -1)[g] = l
                out[at].view(KV, -1, D)[g] = (sc - l[:, None]).exp() @ v
            at += 1
    return {"chosen": torch.from_numpy(chosen).to(DEV), "out": out, "lse": lse, "means": means}


def exact(case, seed):
    st = prepare(case, seed)
    return {"tree": _exact_attention, "weights": _exact_attention, "keep": _exact_keep, "evict": _exact_evict,
            "blocks": _exact_blocks}[case["kind"]](st)
