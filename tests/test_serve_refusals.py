"""What the batch serving operators refuse, before any launch (no GPU needed):
kllm_kv_append, kllm_kv_read, kllm_batch_attention, kllm_sample."""
import ctypes as C

import pytest

A = 1 << 20      # an address on 16 bytes that nothing dereferences: every call here is refused


def _cache(**kw):
    import kmap_b200 as K
    d = dict(format=K.KV_I8, n_seq=2, n_kv=2, head_dim=64, max_pos=16, k=A, v=A, k_scale=A,
             v_scale=A, seq_stride=2 * 16 * 64, scale_stride=2 * 16)
    d.update(kw)
    return K.KvCache(**d)


def _rows(**kw):
    import kmap_b200 as K
    d = dict(rows=1, n_heads=4, pos=A, q=A, k=A, v=A, row_stride=512, head_stride=64, q_out=A)
    d.update(kw)
    return K.KvRows(**d)


def _refused(rc, word):
    import kmap_b200 as K
    msg = K.last_error() or ""
    K.lib().kllm_clear_error()
    assert rc != 0 and word in msg, (rc, msg)


BAD_CACHES = [
    (dict(format=3), "format"), (dict(format=-1), "format"), (dict(head_dim=96), "head dims"),
    (dict(head_dim=0), "head dims"), (dict(n_seq=0), "cache of"), (dict(n_kv=0), "cache of"),
    (dict(max_pos=0), "cache of"), (dict(k=None), "NULL"), (dict(v_scale=None), "NULL"),
    (dict(k=A + 4), "16 bytes"), (dict(seq_stride=2 * 16 * 64 + 8), "16 bytes"),
    (dict(k_scale=A + 2), "scales"), (dict(seq_stride=1024), "overlap"),
    (dict(scale_stride=16), "overlap")]


@pytest.mark.parametrize("kw,word", BAD_CACHES)
def test_bad_caches(built_lib, kw, word):
    import kmap_b200 as K
    c, r = _cache(**kw), _rows()
    _refused(built_lib.kllm_kv_append(C.byref(c), C.byref(r), None), word)
    _refused(built_lib.kllm_kv_read(C.byref(c), 1, None, A, 0, A, A, 128, 64, None), word)
    a = K.BatchAttn(n_seq=2, n_heads=4, max_len=16, scale=1, q=A, q_stride=256,
                    own=C.addressof(c), own_len=A, out=A, out_stride=256, workspace=A,
                    workspace_bytes=1 << 30)
    _refused(built_lib.kllm_batch_attention(C.byref(a), None), word)
    assert built_lib.kllm_batch_attention_workspace(C.byref(a)) == 0
    built_lib.kllm_clear_error()


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "invalid"), (dict(n_heads=-1), "invalid"), (dict(k=None), "invalid"),
    (dict(v=None), "invalid"), (dict(q=None), "invalid"), (dict(q_out=None), "invalid"),
    (dict(rope_cos=A), "together"), (dict(rope_sin=A), "together"),
    (dict(rope_cos=A, rope_sin=A, rope_rows=0), "rope_rows"), (dict(seq=A, pos=None), "seq")])
def test_bad_rows(built_lib, kw, word):
    c, r = _cache(), _rows(**kw)
    _refused(built_lib.kllm_kv_append(C.byref(c), C.byref(r), None), word)


def test_null_arguments(built_lib):
    c, r = _cache(), _rows()
    _refused(built_lib.kllm_kv_append(None, C.byref(r), None), "no cache")
    _refused(built_lib.kllm_kv_append(C.byref(c), None, None), "invalid")
    _refused(built_lib.kllm_kv_read(C.byref(c), 1, None, A, 0, None, A, 128, 64, None), "invalid")
    _refused(built_lib.kllm_kv_read(C.byref(c), -1, None, A, 0, A, A, 128, 64, None), "invalid")
    _refused(built_lib.kllm_kv_read(C.byref(c), 1, A, None, 0, A, A, 128, 64, None), "seq")
    _refused(built_lib.kllm_batch_attention(None, None), "invalid")
    assert built_lib.kllm_batch_attention_workspace(None) == 0
    built_lib.kllm_clear_error()
    _refused(built_lib.kllm_sample(None, None), "invalid")


@pytest.mark.parametrize("kw,word", [
    (dict(n_seq=0), "invalid"), (dict(n_heads=0), "invalid"), (dict(q=None), "invalid"),
    (dict(own=None), "invalid"), (dict(n_heads=5), "5 heads"), (dict(n_seq=3), "own cache"),
    (dict(own_len=None), "own cache"), (dict(max_len=-1), "own cache"),
    (dict(prefix_len=1), "prefix"), (dict(prefix_len=-1), "prefix"), (dict(out=None), "invalid"),
    (dict(workspace=None), "workspace"), (dict(workspace=A + 8), "workspace"),
    (dict(workspace_bytes=16), "workspace"), (dict(q_stride=255), "q_stride"),
    (dict(out_stride=255), "out_stride")])
def test_bad_attention(built_lib, kw, word):
    import kmap_b200 as K
    c = _cache()
    d = dict(n_seq=2, n_heads=4, max_len=16, scale=1, q=A, q_stride=256, own=C.addressof(c),
             own_len=A, out=A, out_stride=256, workspace=A, workspace_bytes=1 << 30)
    d.update(kw)
    a = K.BatchAttn(**d)
    _refused(built_lib.kllm_batch_attention(C.byref(a), None), word)


@pytest.mark.parametrize("kw", [dict(format=2), dict(n_kv=4, seq_stride=4 * 16 * 64, scale_stride=64),
                                dict(head_dim=32)])
def test_caches_that_differ(built_lib, kw):
    import kmap_b200 as K
    c, p = _cache(), _cache(**kw)
    a = K.BatchAttn(n_seq=2, n_heads=4, max_len=16, prefix_len=3, scale=1, q=A, q_stride=256,
                    prefix=C.addressof(p), own=C.addressof(c), own_len=A, out=A, out_stride=256,
                    workspace=A, workspace_bytes=1 << 30)
    _refused(built_lib.kllm_batch_attention(C.byref(a), None), "differ")
    p = _cache()
    a.prefix, a.prefix_len = C.addressof(p), 17
    _refused(built_lib.kllm_batch_attention(C.byref(a), None), "outside")


def test_workspace_size(built_lib):
    """Grows with the rows, needs no device."""
    import kmap_b200 as K
    c = _cache(n_seq=64)
    a = K.BatchAttn(n_seq=1, n_heads=4, max_len=16, scale=1, q=A, q_stride=256,
                    own=C.addressof(c), own_len=A, out=A, out_stride=256)
    one = built_lib.kllm_batch_attention_workspace(C.byref(a))
    a.n_seq = 64
    assert built_lib.kllm_batch_attention_workspace(C.byref(a)) > one > 0


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "invalid"), (dict(vocab=0), "invalid"), (dict(logits=None), "invalid"),
    (dict(u=None), "invalid"), (dict(tokens=None), "invalid"), (dict(row_stride=99), "invalid"),
    (dict(vocab=(1 << 22) + 1, row_stride=1 << 23), "at most")])
def test_bad_sample(built_lib, kw, word):
    import kmap_b200 as K
    d = dict(rows=2, vocab=100, logits=A, row_stride=100, u=A, tokens=A)
    d.update(kw)
    a = K.SampleRows(**d)
    _refused(built_lib.kllm_sample(C.byref(a), None), word)


def test_infer_batch_ex_refuses(built_lib):
    """Before the context is looked at: a format that is none, settings without numbers."""
    import kmap_b200 as K
    one = (C.c_int * 4)(1, 1, 1, 1)
    ctx = built_lib.tape_ctx_create(1, 1)
    for f in (built_lib.kllm_infer_batch_ex, built_lib.kllm_chip_infer_batch_ex):
        _refused(f(None, one, one, 1, 1, -1, None, one, one), "bad argument")
    o = K.BatchOpts(3)
    _refused(built_lib.kllm_infer_batch_ex(ctx, one, one, 1, 1, -1, C.byref(o), one, one), "format")
    o = K.BatchOpts(0, 0, C.addressof(one))
    _refused(built_lib.kllm_infer_batch_ex(ctx, one, one, 1, 1, -1, C.byref(o), one, one), "uniform")
    built_lib.tape_ctx_destroy(ctx)
