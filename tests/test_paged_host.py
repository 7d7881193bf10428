"""What the paged-cache and sampling calls refuse before any launch: bad
shapes, strides, alignments and types, on the host alone (the pointers are
never followed)."""
from __future__ import annotations

import pytest

import grande_amd as g

P = 1 << 20  # an aligned address that is never followed


def kv(**over):
    a = dict(k_ptr=P, v_ptr=P, npages=8, kv_heads=2, page=16, head_dim=64, dtype=g.ELEM_F16)
    a.update(over)
    return g.PagedKv(**a)


def batch(**over):
    a = dict(nseq=3, tokens=3, lens_ptr=P, table_ptr=P, max_pages=4)
    a.update(over)
    return g.PagedBatch(**a)


def source(**over):
    a = dict(dtype=g.ELEM_F32, heads=4, q_ptr=P, k_ptr=P, v_ptr=P, ld=512)
    a.update(over)
    return g.KvSource(**a)


BAD_KV = [(dict(dtype=g.ELEM_F32), "f16 or bf16"), (dict(head_dim=96), "head_dim"), (dict(kv_heads=0), "kv_heads"),
          (dict(page=24), "page"), (dict(npages=0), "npages"), (dict(page_stride=64), "page_stride"),
          (dict(page_stride=16 * 128 + 4), "page_stride"), (dict(k_ptr=P + 2), "aligned"), (dict(v_ptr=None), "aligned")]
BAD_BATCH = [(dict(nseq=0), "nseq"), (dict(tokens=0), "nseq"), (dict(lens_ptr=None), "null"),
             (dict(table_ptr=None), "null"), (dict(tokens=4), "t = nseq"), (dict(max_pages=0), "max_pages"),
             (dict(table_ld=3), "max_pages"), (dict(prefix_len=-1), "prefix_len"), (dict(prefix_len=5), "prefix_table"),
             (dict(max_pages=1 << 28), "max_pages")]


@pytest.mark.parametrize("over,why", BAD_KV)
def test_append_refuses_caches(over, why):
    with pytest.raises(g.OmgError, match=why):
        kv(**over).append(batch(), source(), P, 256)


@pytest.mark.parametrize("over,why", BAD_BATCH)
def test_append_refuses_batches(over, why):
    with pytest.raises(g.OmgError, match=why):
        kv().append(batch(**over), source(), P, 256)


@pytest.mark.parametrize("over,q_out,ldq,why", [
    (dict(dtype=g.ELEM_BF16), P, 256, "cache's type"), (dict(q_ptr=None, k_ptr=None, v_ptr=None), P, 256, "neither"),
    (dict(v_ptr=None), P, 256, "together"), (dict(q_ptr=P + 4), P, 256, "aligned"), (dict(heads=0), P, 256, "heads"),
    (dict(), None, 256, "q_out"), (dict(), P, 252, "ldq"), (dict(), P, 260, "ldq"), (dict(ld=255), P, 256, "ld"),
    (dict(ld=514), P, 256, "ld"), (dict(ldkv=64), P, 256, "ldkv"), (dict(rope=P), P, 256, "rope table"),
    (dict(rope=P, rope_rows=4, rope_dims=24), P, 256, "rope_dims"),
    (dict(rope=P, rope_rows=4, rope_dims=80), P, 256, "rope_dims"),
    (dict(rope=P, rope_rows=4, rope_dims=32, rope_layout=3), P, 256, "layout"),
    (dict(rope=P + 8, rope_rows=4, rope_dims=32), P, 256, "aligned"), (dict(q_norm=P + 4), P, 256, "aligned")])
def test_append_refuses_sources(over, q_out, ldq, why):
    with pytest.raises(g.OmgError, match=why):
        kv().append(batch(), source(**over), q_out, ldq)


def test_append_refuses_null_descriptions():
    import grande_amd._lib as L

    for args in ((None, batch(), source()), (kv(), None, source()), (kv(), batch(), None)):
        with pytest.raises(g.OmgError, match="null"):
            L.check(L.lib().omg_dev_kv_append(*args, P, 256, None))


def attend(k=None, b=None, heads=4, q=P, ldq=256, out=P, ldo=256, scale=0.125, window=0, lse=None, workspace=P,
           workspace_bytes=1 << 40):
    (k or kv()).attention(b or batch(), heads, q, ldq, out, ldo, scale, window=window, lse=lse, workspace=workspace,
                          workspace_bytes=workspace_bytes)


@pytest.mark.parametrize("over,why", BAD_KV)
def test_attention_refuses_caches(over, why):
    with pytest.raises(g.OmgError, match=why):
        attend(k=kv(**over))


@pytest.mark.parametrize("over,why", BAD_BATCH)
def test_attention_refuses_batches(over, why):
    with pytest.raises(g.OmgError, match=why):
        attend(b=batch(**over))


@pytest.mark.parametrize("over,why", [
    (dict(heads=3), "heads"), (dict(heads=0), "heads"), (dict(q=None), "q and out"), (dict(out=P + 2), "q and out"),
    (dict(ldq=248), "ldq"), (dict(ldq=260), "ldq"), (dict(ldo=255), "ldo"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(window=-1), "window"), (dict(b=batch(prefix_table_ptr=P, prefix_len=900), workspace_bytes=16), "workspace needs"),
    (dict(b=batch(prefix_table_ptr=P, prefix_len=900), workspace=None), "workspace must"),
    (dict(b=batch(prefix_table_ptr=P, prefix_len=900), workspace=P + 8), "workspace must")])
def test_attention_refuses_arguments(over, why):
    with pytest.raises(g.OmgError, match=why):
        attend(**over)


def test_workspace_is_refused_or_sized():
    assert kv().attention_workspace(batch(), 4) == 0  # one item a row: no partial results
    assert kv().attention_workspace(batch(prefix_table_ptr=P, prefix_len=900), 4) > 0
    with pytest.raises(g.OmgError, match="heads"):
        kv().attention_workspace(batch(), 3)


@pytest.mark.parametrize("over,why", [
    (dict(dtype=7), "f32, f16 or bf16"), (dict(rows=0), "rows"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 20) + 1, ld=1 << 21), "vocab"), (dict(ld=99), "ld"), (dict(logits_ptr=None), "null"),
    (dict(u_ptr=None), "null"), (dict(tokens_ptr=None), "null"), (dict(logits_ptr=P + 2), "aligned")])
def test_sample_refuses(over, why):
    a = dict(logits_ptr=P, dtype=g.ELEM_F32, rows=3, vocab=100, ld=100, u_ptr=P, tokens_ptr=P)
    a.update(over)
    with pytest.raises(g.OmgError, match=why):
        g.sample(**a, workspace=P, workspace_bytes=1 << 40)


def test_sample_workspace_is_refused_or_sized():
    assert g.sample_workspace(3, 100) >= 0
    for rows, vocab in ((0, 10), (3, 0), (3, (1 << 20) + 1)):
        with pytest.raises(g.OmgError):
            g.sample_workspace(rows, vocab)


def test_calls_past_a_launchs_size_are_refused():
    big = dict(tokens=1 << 24, start_ptr=P)
    with pytest.raises(g.OmgError, match="too many rows"):
        kv().append(batch(**big), source(heads=4096, ld=4096 * 64, ldkv=4096 * 64), P, 4096 * 64)
    with pytest.raises(g.OmgError, match="t \\* heads"):
        attend(b=batch(**big))
    with pytest.raises(g.OmgError, match="too many work items"):
        attend(kv(kv_heads=16), batch(nseq=1 << 20, tokens=1 << 20, start_ptr=P), heads=32, ldq=2048, ldo=2048)
    with pytest.raises(g.OmgError, match="rows must"):
        g.sample_workspace((1 << 21) + 1, 100)
    with pytest.raises(g.OmgError, match="too many logits"):
        g.sample(P, g.ELEM_F16, 1 << 21, 1 << 20, 1 << 20, P, P, workspace=P, workspace_bytes=1 << 60)
