"""How large a call of kllm_batch_attention may be: sizes past what its kernels
count in 32 bits are refused, by the call and by its workspace query alike (no
GPU needed), and a range just below works."""
import ctypes as C

import numpy as np
import pytest

A = 1 << 20      # an address on 16 bytes that nothing dereferences: the calls here are refused


def _call(n_seq, n_heads, max_pos, prefix=False, max_len=None):
    """A call, and the caches that it points to."""
    import kmap_b200 as K
    kv = K.KvCache(K.KV_I8, n_seq, n_heads, 32, max_pos, A, A, A, A, n_heads * max_pos * 32, n_heads * max_pos)
    a = K.BatchAttn(n_seq=n_seq, n_heads=n_heads, scale=1, q=A, q_stride=n_heads * 32, out=A,
                    out_stride=n_heads * 32, workspace=A, workspace_bytes=1 << 62)
    if prefix:
        a.prefix, a.prefix_len = C.addressof(kv), max_pos
    else:
        a.own, a.own_len, a.max_len = C.addressof(kv), A, max_pos if max_len is None else max_len
    return a, kv


@pytest.mark.parametrize("sizes,word", [
    ((1 << 26, 32, 16), "32 bits"),              # query rows
    ((1 << 25, 32, 4096), "blocks"),
    ((1, 1, 0x7fffffff), "32 bits"),             # positions
    ((1, 1, 0x7ffffc01), "32 bits"),
    ((1, 1, 0x7fffffff, True), "32 bits"),
    ((1, 1, 0x7ffffc01, True), "32 bits")])
def test_too_large_is_refused(built_lib, sizes, word):
    import kmap_b200 as K
    a, _kv = _call(*sizes)
    built_lib.kllm_clear_error()
    assert built_lib.kllm_batch_attention(C.byref(a), None) != 0 and word in K.last_error()
    built_lib.kllm_clear_error()
    assert built_lib.kllm_batch_attention_workspace(C.byref(a)) == 0 and word in K.last_error()
    built_lib.kllm_clear_error()


@pytest.mark.parametrize("sizes", [(1, 1, 0x7ffffc00), (1, 1, 0x7ffffc00, True), (64, 1, 0x7ffffc00, True),
                                   (1, 1, 0x7fffffff, False, 100), (1, 1, 100, False, 0x7fffffff)])
def test_large_sizes_have_a_workspace(built_lib, sizes):
    """A few MB for one row, whatever the positions."""
    a, _kv = _call(*sizes)
    assert 0 < built_lib.kllm_batch_attention_workspace(C.byref(a)) < 1 << 30


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_nearly_2_to_31_positions(gpu, n):
    """Every weight is one; the first and last 200 positions alone have values, so
    a lost piece shows.  Keys and values are the same memory (64 GiB)."""
    import torch

    import kmap_b200 as K
    import servecases as S
    hd, P = 32, 0x7ffffc00
    codes = torch.zeros(P, hd, dtype=torch.uint8, device="cuda")
    codes[:200] = 1
    codes[-200:] = 3
    scales = torch.ones(P, device="cuda")
    c = K.KvCache(K.KV_I8, 1, 1, hd, P, codes.data_ptr(), codes.data_ptr(), scales.data_ptr(), scales.data_ptr(),
                  P * hd, P)

    class Prefix:
        pass
    pre = Prefix()
    pre.c = c
    q, out = torch.zeros(n, hd, device="cuda"), torch.zeros(n, hd, device="cuda")
    S.run_attention(q, out, 1, 1.0, pre, P)
    # a part's sums are whole numbers below 2^24 and exact; the join of at most 592 parts, the
    # quotient and exp2 round less than 2^10 times, by 2^-24 at most each
    want = 800 / P
    got = out.cpu().numpy().astype(np.float64)
    del codes, scales
    torch.cuda.empty_cache()
    assert (np.abs(got - want) <= 2.0 ** -14 * want).all()


def test_parts_are_bounded_up_to_the_limit(built_lib):
    """A prefix's parts hold at most 2048 positions (32 floats, a maximum and a sum each)."""
    for P in (1 << 20, 1 << 30, 0x7ffffc00 - 1, 0x7ffffc00):
        a, _kv = _call(1, 1, P, True)
        assert built_lib.kllm_batch_attention_workspace(C.byref(a)) >= (P + 2047) // 2048 * 34 * 4
