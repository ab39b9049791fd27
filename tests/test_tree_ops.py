"""Refusals of the paged append, the paged attention, the tree commit and the
DeltaNet mixer over trees: every check runs on the host before any launch, so
none of the fake pointers below is read. No GPU call is made."""

import pytest

from quicklm_amd import hip

P = 1 << 20  # 16-byte aligned, never dereferenced
ARG, SHAPE = -1, -2


def batch(**kw):
    a = dict(B=2, rows=4, row_start=P, ctx_len=2 * P, parent=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.RowBatch(*a.values())


def pages(**kw):
    a = dict(k=P, v=2 * P, dtype=1, n_pages=8, page_size=16, n_kv=2, hd=128, table=P, ld_table=4)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.KvPages(*a.values())


def append(b=None, p=None, **kw):
    a = dict(qkv=P, ldqkv=2048, qn=P, kn=P, cos=P, sin=P, n_pos=64, rot=32, positions=None,
             ld_pos=0, pair_axis=None, n_axes=1, batch=b or batch(), pages=p or pages(),
             q_out=2 * P, ldq=512, n_q=4, gated=1, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.lib().qlm_paged_append(*a.values())


def attention(b=None, p=None, **kw):
    a = dict(q=P, ldq=512, batch=b or batch(), pages=p or pages(), gate=None, ldg=0, gs=0,
             out=2 * P, ldo=512, n_q=4, work=P, work_bytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.lib().qlm_paged_attention(*a.values())


def commit(b=None, p=None, **kw):
    a = dict(tokens=P, picks=P, batch=b or batch(parent=P), pages=p or pages(), layers=2,
             stride=1 << 20, path=P, ld_path=64, accepted=P, next=P, new_len=P, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.lib().qlm_tree_commit(*a.values())


def tree(b=None, **kw):
    a = dict(proj=P, ldp=1028, batch=b or batch(), conv=P, wt=P, A_log=P, dt=P, norm=P, state=P,
             out=P, ldo=256, H=2, d=128, work=P, work_bytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.lib().qlm_deltanet_tree(*a.values())


def tree_commit(b=None, **kw):
    a = dict(proj=P, ldp=1028, batch=b or batch(), path=P, ld_path=64, accepted=P, conv=P, wt=P,
             A_log=P, dt=P, state=P, H=2, d=128, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return hip.lib().qlm_deltanet_tree_commit(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(row_start=None), ARG), (dict(ctx_len=None), ARG), (dict(B=0), ARG), (dict(B=-1), ARG),
    (dict(rows=0), ARG), (dict(rows=-4), ARG), (dict(B=65536), SHAPE),
    (dict(rows=(1 << 21) + 1), SHAPE),
])
def test_row_batch_refusals(kw, rc):
    for call in (append, attention, tree, tree_commit):
        assert call(batch(**kw)) == rc
    assert commit(batch(**{"parent": P, **kw})) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(table=None), ARG), (dict(dtype=2), ARG),
    (dict(dtype=-1), ARG), (dict(n_pages=0), ARG), (dict(n_kv=0), ARG), (dict(ld_table=0), ARG),
    (dict(page_size=8), SHAPE), (dict(page_size=48), SHAPE), (dict(page_size=512), SHAPE),
    (dict(page_size=0), SHAPE), (dict(hd=64), SHAPE), (dict(hd=192), SHAPE),
    (dict(k=P + 8), SHAPE), (dict(v=P + 2), SHAPE), (dict(ld_table=(1 << 26) + 1), SHAPE),
])
def test_kv_pages_refusals(kw, rc):
    for call in (append, attention, commit):
        assert call(p=pages(**kw)) == rc


def test_missing_structs():
    for call in (append, attention, commit, tree, tree_commit):
        assert call(batch=None) == ARG
    for call in (append, attention, commit):
        assert call(pages=None) == ARG


@pytest.mark.parametrize("kw,rc", [
    (dict(qkv=None), ARG), (dict(q_out=None), ARG), (dict(q_out=P), ARG), (dict(n_q=0), ARG),
    (dict(cos=None), ARG), (dict(sin=None), ARG), (dict(n_pos=0), ARG),
    (dict(positions=P, ld_pos=3), ARG), (dict(positions=P, ld_pos=4, n_axes=0), ARG),
    (dict(rot=31), SHAPE), (dict(rot=-2), SHAPE), (dict(rot=130), SHAPE), (dict(ldq=511), SHAPE),
    (dict(ldqkv=1535), SHAPE), (dict(gated=0, ldqkv=1023), SHAPE), (dict(n_q=8193), SHAPE),
])
def test_append_refusals(kw, rc):
    assert append(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), ARG), (dict(out=None), ARG), (dict(out=P), ARG), (dict(n_q=0), ARG),
    (dict(n_q=3), SHAPE), (dict(n_q=6), SHAPE), (dict(n_q=32, ldq=4096, ldo=4096), SHAPE),
    (dict(ldq=511), SHAPE), (dict(ldo=511), SHAPE), (dict(gate=P, ldg=511, gs=128), SHAPE),
    (dict(gate=P, ldg=2048, gs=127), SHAPE), (dict(work=P + 8), SHAPE),
    (dict(n_q=16, ldq=2048, ldo=2048, gate=P, ldg=2048, gs=1 << 29), SHAPE),  # 15 2^29 > 2^32
])
def test_attention_refusals(kw, rc):
    assert attention(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(tokens=None), ARG), (dict(picks=None), ARG), (dict(path=None), ARG),
    (dict(accepted=None), ARG), (dict(next=None), ARG), (dict(layers=0), ARG),
    (dict(ld_path=63), ARG), (dict(new_len=2 * P), ARG),  # ctx_len itself
    (dict(stride=8 * 2 * 16 * 128 - 1), ARG),  # layers that overlap
    (dict(stride=-1), ARG), (dict(stride=(1 << 20) + 4), SHAPE), (dict(layers=4097), SHAPE),
    (dict(stride=(1 << 48) + 16), SHAPE), (dict(stride=1 << 62), SHAPE),  # bytes past 64 bits
])
def test_commit_refusals(kw, rc):
    assert commit(**kw) == rc


def test_commit_needs_a_tree():
    assert commit(batch()) == ARG


@pytest.mark.parametrize("kw,rc", [
    (dict(proj=None), ARG), (dict(conv=None), ARG), (dict(wt=None), ARG), (dict(A_log=None), ARG),
    (dict(dt=None), ARG), (dict(norm=None), ARG), (dict(state=None), ARG), (dict(out=None), ARG),
    (dict(work=None), ARG), (dict(H=0), ARG), (dict(work_bytes=4 * 256 * 4 - 1), ARG),
    (dict(d=64), SHAPE), (dict(ldp=1027), SHAPE), (dict(ldo=255), SHAPE), (dict(work=P + 4), SHAPE),
    (dict(H=4097, ldp=1 << 22, ldo=1 << 20), SHAPE), (dict(proj=2 * P, out=2 * P), ARG),
])
def test_deltanet_tree_refusals(kw, rc):
    assert tree(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(proj=None), ARG), (dict(path=None), ARG), (dict(accepted=None), ARG),
    (dict(conv=None), ARG), (dict(state=None), ARG), (dict(ld_path=0), ARG), (dict(d=256), SHAPE),
    (dict(ldp=1027), SHAPE),
])
def test_deltanet_tree_commit_refusals(kw, rc):
    assert tree_commit(**kw) == rc


@pytest.mark.parametrize("rows,B,n_q,n_kv,hd,slots", [
    (1, 1, 16, 4, 128, 1040), (512, 8, 16, 4, 128, 4096), (2048, 1, 16, 2, 256, 32768),
    (64, 64, 8, 8, 128, 8192)])
def test_attention_workspace(rows, B, n_q, n_kv, hd, slots):
    L = hip.lib()
    n = L.qlm_paged_attention_workspace_bytes(rows, B, n_q, n_kv, hd, slots)
    assert n > 0
    kw = dict(b=batch(B=B, rows=rows), p=pages(n_kv=n_kv, hd=hd, ld_table=slots // 16), n_q=n_q,
              ldq=n_q * hd, ldo=n_q * hd)
    assert attention(work_bytes=n - 1, **kw) == ARG
    assert attention(work=None, **kw) == ARG
    for bad in [(0, B, n_q, n_kv, hd, slots), (rows, 0, n_q, n_kv, hd, slots),
                (rows, B, n_q + 1, n_kv, hd, slots), (rows, B, n_q, n_kv, 64, slots),
                (rows, B, n_q, n_kv, hd, 0), (rows, B, 16 * n_kv, n_kv, hd, slots)]:
        assert L.qlm_paged_attention_workspace_bytes(*bad) == 0


def test_attention_without_a_workspace():
    """Few rows and few slots: nothing is cut, nothing joined."""
    assert hip.lib().qlm_paged_attention_workspace_bytes(4, 4, 16, 4, 128, 1024) == 0


def test_deltanet_tree_workspace():
    q = hip.lib().qlm_deltanet_tree_workspace_bytes
    assert q(4, 2, 128) > 0
    for bad in [(0, 2, 128), (4, 0, 128), (4, 2, 64), ((1 << 21) + 1, 2, 128), (4, 4097, 128)]:
        assert q(*bad) == 0
