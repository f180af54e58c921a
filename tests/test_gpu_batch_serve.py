"""The batch serving operators together, as kllm_chip_infer_batch_ex runs
them: prompts with a common prefix, caches in 8 bits, drawn tokens.

With fp32 caches every sequence's tokens equal the oracle's single-sequence
run, prefix or not.  A drawn token is checked against the definition on the
logits that the fused single-sequence run has at that step, where the number
is far enough from a border that the logits' tolerance cannot matter.  8-bit
caches change the logits: a shared prefix has to give the tokens that one
stored per sequence gives."""
import dataclasses

import numpy as np
import pytest

import harness

pytestmark = pytest.mark.gpu


def _prompts(V, lens, shared, seed):
    rng = np.random.default_rng(seed)
    head = rng.integers(3, V, shared).astype(np.int32)
    return [np.concatenate([head, rng.integers(3, V, n).astype(np.int32)]) for n in lens]


@pytest.mark.parametrize("name", ["gqa", "mha", "tl"])
@pytest.mark.parametrize("tc", ["1", "0"])
@pytest.mark.parametrize("shared,lens", [(0, [1, 5, 3]), (1, [1, 4]), (20, [1, 9, 4, 2, 1]),
                                         (17, [0, 0, 0]), (30, [0, 6])])
def test_shared_prefix_keeps_the_oracles_tokens(gpu, oracle, chip_dir, name, tc, shared, lens,
                                                monkeypatch):
    """fp32 caches.  Equal prompts and prompts that are each other's beginnings
    keep their last token out of the prefix."""
    import kmap_b200
    monkeypatch.setenv("KLLM_BATCH_TC", tc)
    path, max_new = chip_dir(name), 10
    with kmap_b200.Chip(path) as chip:
        prompts = [p for p in _prompts(chip.info["vocab_size"], lens, shared, 3) if len(p)]
        outs = chip.infer_batch(prompts, max_new, share_prefix=True)
        held = chip.stats()["shared_prefix"]
        again = chip.infer_batch(prompts, max_new, share_prefix=True, use_graphs=False)
    common = min(len(p) for p in prompts) - 1
    while any((p[:common] != prompts[0][:common]).any() for p in prompts):
        common -= 1
    assert held == common >= min(shared, common)
    assert [o.tolist() for o in again] == [o.tolist() for o in outs]
    oc = harness.OracleChip(oracle, path)
    for p, toks in zip(prompts, outs):
        assert toks.tolist() == oc.infer(p, max_new)[0].tolist()
    oc.close()


@pytest.mark.parametrize("fmt", ["f32", "i8", "e4m3"])
@pytest.mark.parametrize("share", [False, True])
def test_drawn_tokens(gpu, chip_dir, fmt, share):
    """Same numbers, same tokens: with and without the graph, whatever the order of
    the sequences; greedy settings draw what the greedy run picks; top_k = 1 too."""
    import kmap_b200 as K
    kf = {"f32": K.KV_F32, "i8": K.KV_I8, "e4m3": K.KV_E4M3}[fmt]
    path, n, new = chip_dir("tl"), 6, 12
    u = np.random.default_rng(5).random((n, new)).astype(np.float32)
    with K.Chip(path) as chip:
        prompts = _prompts(chip.info["vocab_size"], [1, 5, 2, 7, 1, 3], 25, 4)
        kw = dict(kv_format=kf, share_prefix=share)
        a = chip.infer_batch(prompts, new, u=u, temperature=0.9, top_k=50, top_p=0.95, min_p=0.01, **kw)
        b = chip.infer_batch(prompts, new, u=u, temperature=0.9, top_k=50, top_p=0.95, min_p=0.01,
                             use_graphs=False, **kw)
        c = chip.infer_batch(prompts[::-1], new, u=u[::-1], temperature=0.9, top_k=50, top_p=0.95,
                             min_p=0.01, **kw)
        greedy = chip.infer_batch(prompts, new, **kw)
        cold = chip.infer_batch(prompts, new, u=u, temperature=0.0, **kw)
        one = chip.infer_batch(prompts, new, u=u, top_k=np.ones(n), **kw)
    t = lambda x: [o.tolist() for o in x]
    assert t(a) == t(b) == t(c)[::-1]
    assert t(greedy) == t(cold) == t(one)
    assert t(a) != t(greedy)


def test_draws_follow_the_definition(gpu, chip_dir):
    """Each drawn token against the plain definition on the logits of the fused
    single-sequence run of the same tokens (within 1e-3 of the batch's): equal
    wherever numbers 1 % to either side draw the same token."""
    import kmap_b200 as K
    import servecases as S
    path, n, new = chip_dir("gqa"), 8, 8
    rng = np.random.default_rng(9)
    u = rng.random((n, new)).astype(np.float32)
    T = np.float32(0.7)
    checked = 0
    with K.Chip(path) as chip:
        prompts = _prompts(chip.info["vocab_size"], [2] * n, 20, 6)
        outs = chip.infer_batch(prompts, new, u=u, temperature=T, top_k=20, share_prefix=True)
        for i, (p, toks) in enumerate(zip(prompts, outs)):
            full = np.concatenate([p, toks]).astype(np.int32)
            _, lg = chip.infer(full, 1, logits=True)
            for j in range(new):
                row = lg[len(p) - 1 + j]
                near = {S.sample_plain(row, float(T), 20, 1.0, 0.0, float(u[i, j]) + d)
                        for d in (-0.01, -0.005, 0.0, 0.005, 0.01)}
                if len(near) == 1:
                    checked += 1
                    assert toks[j] == near.pop()
    assert checked > n * new // 3


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_eight_bit_caches(gpu, chip_dir, fmt):
    """A prefix that is shared or stored once per sequence gives the same tokens:
    the prefix's stored values are what every later position attends to.  Without
    sharing a prompt's positions see each other in fp32, so only the single token
    behind the prefix (the first decoded position) can be compared: its keys are
    the stored ones in both."""
    import kmap_b200 as K
    kf = {"i8": K.KV_I8, "e4m3": K.KV_E4M3}[fmt]
    path, new = chip_dir("tl"), 8
    with K.Chip(path) as chip:
        # every prompt is the prefix and one token of its own
        prompts = _prompts(chip.info["vocab_size"], [1] * 5, 40, 8)
        a = chip.infer_batch(prompts, new, kv_format=kf, share_prefix=True)
        assert chip.stats()["shared_prefix"] == 40
        b = chip.infer_batch(prompts, new, kv_format=kf)
        assert chip.stats()["shared_prefix"] == 0
        # EOS cuts
        eos = int(a[2][3])
        cut = chip.infer_batch(prompts, new, eos=eos, kv_format=kf, share_prefix=True)
    assert [x.tolist() for x in a] == [x.tolist() for x in b]
    for f, c in zip(a, cut):
        k = int(np.nonzero(f == eos)[0][0]) if (f == eos).any() else len(f)
        assert c.tolist() == f[:k].tolist()


def test_plain_calls_are_unchanged_between(gpu, chip_dir):
    """The prompt passes of a serving batch use the single-sequence cache: a
    single-sequence call after one gives what it gave before."""
    import kmap_b200 as K
    path = chip_dir("gqa")
    with K.Chip(path) as chip:
        V = chip.info["vocab_size"]
        prompts = _prompts(V, [3, 1, 4], 15, 2)
        one = chip.infer(prompts[0], 8).tolist()
        plain = [o.tolist() for o in chip.infer_batch(prompts, 8)]
        chip.infer_batch(prompts, 8, kv_format=K.KV_I8, share_prefix=True)
        assert chip.infer(prompts[0], 8).tolist() == one
        assert [o.tolist() for o in chip.infer_batch(prompts, 8)] == plain


def test_tinyllama_width_matches_reference(gpu, ref, tmp_path):
    import kmap_b200
    from kmap_b200 import chipgen
    spec = dataclasses.replace(chipgen.TINYLLAMA_1B, num_layers=2, max_seq=256)
    path = chipgen.ensure_chip(str(tmp_path), spec)
    prompts = _prompts(spec.vocab_size, [1, 9, 30], 150, 17)
    with kmap_b200.Chip(path) as chip:
        outs = chip.infer_batch(prompts, 8, share_prefix=True)
        assert chip.stats()["shared_prefix"] == 150
    h, info = ref.chip(path)
    for p, toks in zip(prompts, outs):
        assert toks.tolist() == ref.infer(h, p, 8).tolist()
    ref.L.refh_chip_destroy(h)


def test_wrong_numbers_are_refused(gpu, chip_dir):
    import kmap_b200 as K
    with K.Chip(chip_dir("gqa")) as chip:
        with pytest.raises(K.KllmError, match="shape"):
            chip.infer_batch([[5, 6]], 4, u=np.zeros((1, 3)))
        with pytest.raises(K.KllmError, match="uniform"):
            chip.infer_batch([[5, 6]], 4, temperature=0.5)
        with pytest.raises(K.KllmError, match="format"):
            chip.infer_batch([[5, 6]], 4, kv_format=7)
