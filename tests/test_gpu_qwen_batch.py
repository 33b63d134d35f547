"""QwenDecoder.generate_batch: every prompt's ids are those that generate()
selects for it alone, whatever else is in flight -- more prompts than places,
prompts longer than a step, prompts that end at different steps -- and the
decoder's own sequence is left as it was."""
import os

import numpy as np
import pytest

from conftest import CACHE, golden, mit2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qwen(gpt_mod):
    g = golden("qwen.npz")
    path = os.path.join(CACHE, "qwen_s44_g20")
    assert mit2.write_synthetic_qwen_bundle(path, seed=int(g["bundle_seed"]),
                                            eos_gain=float(g["bundle_eos_gain"])) == str(g["bundle_sha256"])
    d = gpt_mod.QwenDecoder(path)
    yield d
    d.close()


@pytest.mark.parametrize("names", ["a", "b", "ab", "bababbaaabababbababaab"])
def test_batch_matches_reference(qwen, names):
    g = golden("qwen.npz")
    got = qwen.generate_batch([g[f"{n}.ids"] for n in names], 128)
    assert len(got) == len(names)
    for n, r in zip(names, got):
        assert r.stopped
        np.testing.assert_array_equal(r.codes, g[f"{n}.generated"])
    t = qwen.last_timing()
    assert t.prompt == sum(g[f"{n}.ids"].size for n in names) and t.decode_ms > 0
    assert t.steps >= max(g[f"{n}.generated"].size for n in names)


def selections(qwen, ids, count):
    """The ids that the decoder selects one by one, up to the first that is not 1e-3 ahead of the next."""
    lg = qwen.prefill(ids)
    out = []
    for _ in range(count):
        top = np.partition(lg, -2)[-2:]
        if top[1] - top[0] < 1e-3:
            break
        out.append(int(np.argmax(lg)))
        lg = qwen.step(out[-1])
    return out


def test_prompts_longer_than_a_step(qwen):
    """1500 and 2500 ids take two and three steps, beside prompts that generate meanwhile."""
    g = golden("qwen.npz")
    r = np.random.default_rng(11)
    prompts = [r.integers(0, 151000, n).astype(np.uint32) for n in (1500, 1, 2500, 64, 65)]
    want = [selections(qwen, p, 4) for p in prompts]
    assert sum(map(len, want)) >= 10
    got = qwen.generate_batch(prompts + [g["a.ids"]], 24)
    for w, x in zip(want, got):
        assert list(x.codes[:len(w)]) == w[:x.codes.size]
        assert x.stopped == (x.codes[-1] == 151643) and (x.stopped or x.codes.size == 24)
    np.testing.assert_array_equal(got[-1].codes, g["a.generated"])


def test_a_run_without_eos_is_not_stopped(qwen):
    g = golden("qwen.npz")
    want = g["b.generated"]
    a, b, c = qwen.generate_batch([g["a.ids"], g["b.ids"], g["b.ids"]], 20)
    assert a.stopped and not b.stopped and not c.stopped
    np.testing.assert_array_equal(b.codes, want[:20])
    np.testing.assert_array_equal(c.codes, want[:20])
    (one,) = qwen.generate_batch([g["b.ids"]], 1)
    assert list(one.codes) == [want[0]] and not one.stopped


def test_the_decoders_own_sequence_is_kept(qwen):
    g = golden("qwen.npz")
    qwen.prefill(g["b.ids"])
    want = qwen.step(int(g["b.generated"][0]))
    qwen.prefill(g["b.ids"])
    qwen.generate_batch([g["a.ids"]] * 3, 16)
    assert qwen.cached_tokens() == g["b.ids"].size
    np.testing.assert_array_equal(qwen.step(int(g["b.generated"][0])), want)
    np.testing.assert_array_equal(qwen.generate(g["a.ids"], 128), g["a.generated"])


def test_errors(qwen):
    ok = np.array([1, 2], np.uint32)
    assert qwen.generate_batch([], 8) == []
    for bad, maximum, text in (([], 8, "Qwen prompt capacity is 3072 tokens"),
                               (np.zeros(3073, np.uint32), 8, "Qwen prompt capacity is 3072 tokens"),
                               (np.array([151936], np.uint32), 8, "Invalid Qwen token"),
                               (ok, 0, "Qwen generation capacity exceeded"),
                               (ok, 1025, "Qwen generation capacity exceeded"),
                               (np.zeros(3500, np.uint32), 700, "Qwen generation capacity exceeded")):
        with pytest.raises(ValueError, match=text):
            qwen.generate_batch([ok, bad], maximum)
