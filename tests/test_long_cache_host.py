"""What the calls for long caches (tree attention, moved rows, attention
weights, eviction, attention over chosen blocks) refuse before any launch, on
the host alone (the pointers are never followed)."""
from __future__ import annotations

import pytest

import grande_amd as g
from test_paged_host import BAD_BATCH, BAD_KV, P, batch, kv

NAN, INF = float("nan"), float("inf")


def tree(k=None, b=None, heads=4, q=P, ldq=256, out=P, ldo=256, scale=0.125, mask=P, mask_ld=1, workspace=P,
         workspace_bytes=1 << 40, **kw):
    (k or kv()).attention_tree(b or batch(), heads, q, ldq, out, ldo, scale, mask, mask_ld, workspace=workspace,
                               workspace_bytes=workspace_bytes, **kw)


LONG = dict(prefix_table_ptr=P, prefix_len=900)
ROWS = [(dict(heads=3), "heads"), (dict(heads=0), "heads"), (dict(heads=8192), "heads"), (dict(q=None), "q and out"),
        (dict(out=P + 2), "q and out"), (dict(ldq=248), "ldq"), (dict(ldq=260), "ldq"), (dict(ldo=255), "ldo"),
        (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=NAN), "scale"), (dict(scale=INF), "scale")]


@pytest.mark.parametrize("over,why", BAD_KV)
def test_tree_refuses_caches(over, why):
    with pytest.raises(g.OmgError, match=f"attention_tree.*{why}"):
        tree(k=kv(**over))


@pytest.mark.parametrize("over,why", BAD_BATCH)
def test_tree_refuses_batches(over, why):
    with pytest.raises(g.OmgError, match=f"attention_tree.*{why}"):
        tree(b=batch(**over))


@pytest.mark.parametrize("over,why", ROWS + [
    (dict(mask=None), "mask"), (dict(mask=P + 2), "mask"), (dict(mask_ld=0), "mask_ld"), (dict(mask_ld=-1), "mask_ld"),
    (dict(mask_ld=(1 << 20) + 1), "mask_ld"), (dict(window=-1), "window"), (dict(window=5), "positions"),
    (dict(window=5, positions=P + 2), "positions"), (dict(b=batch(**LONG), workspace_bytes=16), "workspace needs"),
    (dict(b=batch(**LONG), workspace=None), "workspace must"), (dict(b=batch(**LONG), workspace=P + 8), "workspace must")])
def test_tree_refuses_arguments(over, why):
    with pytest.raises(g.OmgError, match=f"attention_tree.*{why}"):
        tree(**over)


def test_tree_workspace_is_refused_or_sized():
    assert kv().attention_tree_workspace(batch(), 4) == 0
    assert kv().attention_tree_workspace(batch(**LONG), 4) == kv().attention_workspace(batch(**LONG), 4)
    with pytest.raises(g.OmgError, match="attention_tree.*heads"):
        kv().attention_tree_workspace(batch(), 3)


def test_tree_refuses_null_descriptions():
    import grande_amd._lib as L

    for args in ((None, batch()), (kv(), None)):
        with pytest.raises(g.OmgError, match="null"):
            L.check(L.lib().omg_dev_attention_tree(*args, 4, P, 256, P, 256, None, 0.125, P, 1, 0, None, P, 1 << 40, None))


def keep(k=None, b=None, rows=P, rows_ld=8, count=8, **kw):
    (k or kv()).keep(b or batch(), rows, rows_ld, count, **kw)


@pytest.mark.parametrize("over,why", BAD_KV)
def test_keep_and_evict_refuse_caches(over, why):
    with pytest.raises(g.OmgError, match=f"kv_keep.*{why}"):
        keep(k=kv(**over))
    with pytest.raises(g.OmgError, match=f"kv_evict.*{why}"):
        evict(k=kv(**over))


@pytest.mark.parametrize("over,why", [x for x in BAD_BATCH if "prefix_len" not in x[0]])
def test_keep_and_evict_refuse_batches(over, why):
    with pytest.raises(g.OmgError, match=f"kv_keep.*{why}"):
        keep(b=batch(**over))
    with pytest.raises(g.OmgError, match=f"kv_evict.*{why}"):
        evict(b=batch(**over))


@pytest.mark.parametrize("over,why", [
    (dict(rows=None), "null rows"), (dict(count=0), "count"), (dict(count=65, rows_ld=65), "count"),
    (dict(rows_ld=7), "rows_ld"), (dict(to_table=P, to_ld=0), "to_ld"), (dict(to_table=P, to_ld=1 << 28), "to_ld")])
def test_keep_refuses_arguments(over, why):
    with pytest.raises(g.OmgError, match=f"kv_keep.*{why}"):
        keep(**over)


def evict(k=None, b=None, keep=20, recent=5, weights=P, ldw=64, rows=P, **kw):
    (k or kv()).evict(b or batch(), keep, recent, weights, ldw, rows, **kw)


@pytest.mark.parametrize("over,why", [
    (dict(weights=None), "null"), (dict(rows=None), "null"), (dict(keep=0), "keep"), (dict(recent=-1), "recent"),
    (dict(recent=21), "recent"), (dict(keep=65), "sequence's rows"), (dict(ldw=63), "ldw"),
    (dict(kept_weights=P + 4096, kept_ld=19), "kept_ld"), (dict(to_table=P, to_ld=0), "to_ld"),
    (dict(to_table=P, to_ld=1 << 28), "to_ld")])
def test_evict_refuses_arguments(over, why):
    with pytest.raises(g.OmgError, match=f"kv_evict.*{why}"):
        evict(**over)


def test_keep_and_evict_refuse_null_descriptions_and_too_many_lists():
    import grande_amd._lib as L

    for args in ((None, batch()), (kv(), None)):
        with pytest.raises(g.OmgError, match="null"):
            L.check(L.lib().omg_dev_kv_keep(*args, P, 8, 8, None, 0, None, 0, None))
        with pytest.raises(g.OmgError, match="null"):
            L.check(L.lib().omg_dev_kv_evict(*args, 20, 5, P, 64, P, None, 0, None, 0, None))
    many = batch(nseq=1 << 20, tokens=1 << 20)
    with pytest.raises(g.OmgError, match="kv_keep: too many lists"):
        keep(k=kv(kv_heads=64), b=many)
    with pytest.raises(g.OmgError, match="kv_keep: too many rows"):
        keep(k=kv(kv_heads=64), b=many, count=64, rows_ld=64, to_table=P, to_ld=4)
    with pytest.raises(g.OmgError, match="kv_evict: too many lists"):
        evict(k=kv(kv_heads=64), b=many)


def weigh(k=None, b=None, heads=4, q=P, ldq=256, lse=P, scale=0.125, weights=P, ldw=64, workspace=P,
          workspace_bytes=1 << 40, **kw):
    (k or kv()).attention_weights(b or batch(), heads, q, ldq, lse, scale, weights, ldw, workspace=workspace,
                                  workspace_bytes=workspace_bytes, **kw)


@pytest.mark.parametrize("over,why", BAD_KV)
def test_weights_refuse_caches(over, why):
    with pytest.raises(g.OmgError, match=f"attention_weights.*{why}"):
        weigh(k=kv(**over))


@pytest.mark.parametrize("over,why", BAD_BATCH)
def test_weights_refuse_batches(over, why):
    with pytest.raises(g.OmgError, match=f"attention_weights.*{why}"):
        weigh(b=batch(**over))


PROMPT = dict(nseq=1, tokens=4000, start_ptr=P, max_pages=300)


@pytest.mark.parametrize("over,why", [
    (dict(heads=3), "heads"), (dict(heads=0), "heads"), (dict(q=None), "q must"), (dict(q=P + 2), "q must"),
    (dict(ldq=248), "ldq"), (dict(ldq=260), "ldq"), (dict(ldq=(1 << 24) + 8), "ldq"), (dict(lse=None), "null"), (dict(weights=None), "null"),
    (dict(ldw=63), "ldw"), (dict(scale=0.0), "scale"), (dict(scale=NAN), "scale"), (dict(scale=INF), "scale"),
    (dict(window=-1), "window"), (dict(b=batch(**PROMPT), ldw=4800, workspace_bytes=16), "workspace needs"),
    (dict(b=batch(**PROMPT), ldw=4800, workspace=None), "workspace must"),
    (dict(b=batch(**PROMPT), ldw=4800, workspace=P + 8), "workspace must")])
def test_weights_refuse_arguments(over, why):
    with pytest.raises(g.OmgError, match=f"attention_weights.*{why}"):
        weigh(**over)


def test_weights_workspace_and_sizes():
    assert kv().attention_weights_workspace(batch(), 4) == 0
    assert kv().attention_weights_workspace(batch(**PROMPT), 4) > 0
    with pytest.raises(g.OmgError, match="attention_weights.*heads"):
        kv().attention_weights_workspace(batch(), 3)
    with pytest.raises(g.OmgError, match="t \\* heads"):
        weigh(b=batch(tokens=1 << 24, start_ptr=P))
    with pytest.raises(g.OmgError, match="too many work items"):
        weigh(k=kv(kv_heads=32), b=batch(nseq=1 << 20, tokens=1 << 20), heads=32, ldq=2048)


def blocks(k=None, b=None, heads=4, q=P, ldq=256, out=P, ldo=256, scale=0.125, means=P, blocks=4, workspace=P,
           workspace_bytes=1 << 40, **kw):
    (k or kv()).attention_blocks(b or batch(), heads, q, ldq, out, ldo, scale, means, blocks, workspace=workspace,
                                 workspace_bytes=workspace_bytes, **kw)


@pytest.mark.parametrize("over,why", BAD_KV)
def test_blocks_refuse_caches(over, why):
    with pytest.raises(g.OmgError, match=f"attention_blocks.*{why}"):
        blocks(k=kv(**over))
    with pytest.raises(g.OmgError, match=f"block_means.*{why}"):
        kv(**over).block_means(batch(), P)


@pytest.mark.parametrize("over,why", BAD_BATCH)
def test_blocks_refuse_batches(over, why):
    with pytest.raises(g.OmgError, match=f"attention_blocks.*{why}"):
        blocks(b=batch(**over))
    with pytest.raises(g.OmgError, match=f"block_means.*{why}"):
        kv().block_means(batch(**over), P)


@pytest.mark.parametrize("over,why", ROWS + [
    (dict(means=None), "means"), (dict(means=P + 8), "means"), (dict(blocks=0), "blocks must"), (dict(blocks=4097), "blocks must"),
    (dict(workspace_bytes=16), "workspace needs"), (dict(workspace=None), "workspace must"),
    (dict(workspace=P + 8), "workspace must")])
def test_blocks_refuse_arguments(over, why):
    with pytest.raises(g.OmgError, match=f"attention_blocks.*{why}"):
        blocks(**over)


def test_blocks_workspace_and_sizes():
    assert kv().attention_blocks_workspace(batch(), 4, 2) > 0
    for heads, n in ((3, 2), (4, 0), (4, 4097)):
        with pytest.raises(g.OmgError, match="attention_blocks"):
            kv().attention_blocks_workspace(batch(), heads, n)
    for means in (None, P + 4):
        with pytest.raises(g.OmgError, match="block_means: means"):
            kv().block_means(batch(), means)
    with pytest.raises(g.OmgError, match="too many rows"):
        kv(kv_heads=64).block_means(batch(nseq=1 << 20, tokens=1 << 20), P)
    with pytest.raises(g.OmgError, match="t \\* heads"):
        blocks(b=batch(tokens=1 << 24, start_ptr=P))
    with pytest.raises(g.OmgError, match="too many work items"):
        blocks(k=kv(kv_heads=32), b=batch(nseq=1 << 20, tokens=1 << 20), heads=32, ldq=2048, ldo=2048, workspace_bytes=1 << 60)


def test_blocks_and_weights_refuse_null_descriptions():
    import grande_amd._lib as L

    for args in ((None, batch()), (kv(), None)):
        for call in (lambda: L.lib().omg_dev_block_means(*args, P, None),
                     lambda: L.lib().omg_dev_attention_blocks(*args, 4, P, 256, P, 256, None, 0.125, P, 4, None, P, 1 << 40, None),
                     lambda: L.lib().omg_dev_attention_weights(*args, 4, P, 256, P, 0.125, 0, P, 64, P, 1 << 40, None)):
            with pytest.raises(g.OmgError, match="null"):
                L.check(call())
