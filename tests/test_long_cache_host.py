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
