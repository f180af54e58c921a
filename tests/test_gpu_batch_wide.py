"""kllm_chip_infer_batch_ex where the shared prefix goes through the tiles of
128 query rows: 48 sequences of 8 heads of 32 on 2 kv heads (192 query rows of
a kv head) behind a long prompt."""
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
