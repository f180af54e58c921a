"""kllm_chip_infer_batch_ex where the shared prefix goes through the tiles of
128 query rows: 48 sequences of 8 heads of 32 on 2 kv heads (192 query rows of
a kv head) behind a long prompt; and at a width where the projections come as
sums of several partial planes."""
import dataclasses

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wide_chip(tmp_path_factory):
    from kmap_b200 import chipgen
    made = {}

    def get(max_seq):
        if max_seq not in made:
            spec = chipgen.ModelSpec(num_layers=2, hidden_size=256, num_attention_heads=8,
                                     num_key_value_heads=2, intermediate_size=512, vocab_size=600,
                                     max_seq=max_seq, norm_weights="random", seed=11)
            made[max_seq] = chipgen.ensure_chip(str(tmp_path_factory.mktemp("wide")), spec)
        return made[max_seq]
    return get


def _prompts(n, shared, V=600, seed=1):
    rng = np.random.default_rng(seed)
    head = rng.integers(3, V, shared).astype(np.int32)
    return [np.concatenate([head, np.array([3 + i], np.int32)]) for i in range(n)]


def test_a_wait_that_gives_up_is_an_error(gpu, wide_chip, monkeypatch):
    """With a limit of 0 the first wait that would have to wait gives up: the call
    returns the status instead of tokens, and the next call runs as before."""
    import kmap_b200 as K
    prompts = _prompts(48, 1040)
    with K.Chip(wide_chip(1100)) as chip:
        kw = dict(kv_format=K.KV_I8, share_prefix=True)
        want = [o.tolist() for o in chip.infer_batch(prompts, 4, **kw)]
        assert chip.stats()["shared_prefix"] == 1040
        monkeypatch.setenv("KLLM_WAIT_LIMIT_MS", "0")
        for graphs in (True, False):
            with pytest.raises(K.KllmError, match="status.*timed out"):
                chip.infer_batch(prompts, 4, use_graphs=graphs, **kw)
        monkeypatch.delenv("KLLM_WAIT_LIMIT_MS")
        assert [o.tolist() for o in chip.infer_batch(prompts, 4, **kw)] == want


@pytest.mark.parametrize("fmt,shared", [("i8", 1040), ("e4m3", 1040), ("f32", 2700)])
@pytest.mark.parametrize("tc", ["1", "0"])
def test_128_row_tiles_give_the_same_tokens(gpu, wide_chip, fmt, shared, tc, monkeypatch):
    """Each prompt is the prefix and one token, so with 8 bits too the keys and values that a
    decoded position sees are the same ones, read once or stored per sequence."""
    import kmap_b200 as K
    monkeypatch.setenv("KLLM_BATCH_TC", tc)
    kf = {"f32": K.KV_F32, "i8": K.KV_I8, "e4m3": K.KV_E4M3}[fmt]
    prompts = _prompts(48, shared)
    with K.Chip(wide_chip(shared + 60)) as chip:
        a = chip.infer_batch(prompts, 6, kv_format=kf, share_prefix=True)
        assert chip.stats()["shared_prefix"] == shared
        b = chip.infer_batch(prompts, 6, kv_format=kf)
        assert chip.stats()["shared_prefix"] == 0
    assert [x.tolist() for x in a] == [x.tolist() for x in b]
    assert len({tuple(x.tolist()) for x in a}) > 24      # (the sequences do differ)


def test_partial_planes_at_a_models_width(gpu, tmp_path):
    """TinyLlama's widths, two layers: the projections' K ranges come as several planes, whose sum the
    append and the draw take.  Greedy tokens equal those of the plain batch (its own kernels), and
    drawn ones the definition on the logits of the single-sequence run, where numbers 1 % to either
    side draw the same."""
    import kmap_b200 as K
    import servecases as S
    from kmap_b200 import chipgen
    spec = dataclasses.replace(chipgen.TINYLLAMA_1B, num_layers=2, max_seq=256)
    path = chipgen.ensure_chip(str(tmp_path), spec)
    rng = np.random.default_rng(17)
    head = rng.integers(3, spec.vocab_size, 60).astype(np.int32)
    prompts = [np.concatenate([head, rng.integers(3, spec.vocab_size, m).astype(np.int32)]) for m in (1, 9, 30, 2, 5)]
    n, new = len(prompts), 6
    u = rng.random((n, new)).astype(np.float32)
    T = np.float32(0.8)
    checked = 0
    with K.Chip(path) as chip:
        plain = [x.tolist() for x in chip.infer_batch(prompts, new)]
        assert [x.tolist() for x in chip.infer_batch(prompts, new, share_prefix=True)] == plain
        assert chip.stats()["shared_prefix"] >= 60
        cold = chip.infer_batch(prompts, new, share_prefix=True, u=u, temperature=0.0)
        assert [x.tolist() for x in cold] == plain
        drawn = chip.infer_batch(prompts, new, share_prefix=True, u=u, temperature=T, top_k=30, top_p=0.9)
        for i, (p, toks) in enumerate(zip(prompts, drawn)):
            _, lg = chip.infer(np.concatenate([p, toks]).astype(np.int32), 1, logits=True)
            for j in range(new):
                row = lg[len(p) - 1 + j]
                near = {S.sample_plain(row, float(T), 30, float(np.float32(0.9)), 0.0, float(u[i, j]) + d)
                        for d in (-0.01, -0.005, 0.0, 0.005, 0.01)}
                if len(near) == 1:
                    checked += 1
                    assert toks[j] == near.pop()
    assert checked > n * new // 3


def test_a_wait_that_gives_up_with_fp32_caches(gpu, wide_chip, monkeypatch):
    """As above, for the kernel that feeds keys and values by warps of their own."""
    import kmap_b200 as K
    prompts = _prompts(48, 2700)
    with K.Chip(wide_chip(2760)) as chip:
        want = [o.tolist() for o in chip.infer_batch(prompts, 3, share_prefix=True)]
        monkeypatch.setenv("KLLM_WAIT_LIMIT_MS", "0")
        with pytest.raises(K.KllmError, match="status.*timed out"):
            chip.infer_batch(prompts, 3, share_prefix=True)
        monkeypatch.delenv("KLLM_WAIT_LIMIT_MS")
        assert [o.tolist() for o in chip.infer_batch(prompts, 3, share_prefix=True)] == want
