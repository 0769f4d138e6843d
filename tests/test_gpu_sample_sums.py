"""What gh_sample_rows holds of weights and sums, at the largest vocabularies, and rows just as long as its list and longer."""
import numpy as np
import pytest

import flat_tail
from test_gpu_sample import SETTINGS, check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,distance", [(131072, 23.5), ((1 << 17) + 1, 23.5), (1 << 20, 25.5), (1 << 24, 27.5), (1 << 24, 26.9)])
def test_a_flat_far_tail_keeps_its_mass(hip, vocab, distance):
    def by_batch(logits, want, us):
        got = [run(hip, logits, [c[0] for c in want[i:i + len(us)]], us) for i in range(0, len(want), len(us))]
        return np.concatenate([g[0] for g in got]), np.concatenate([g[1] for g in got])
    flat_tail.check(by_batch, vocab, distance)


@pytest.mark.parametrize("vocab", [7679, 7680, 7681])
def test_as_many_tokens_as_the_list_takes(hip, rng, vocab):
    logits = (7 + 0.0005 * rng.random((8, vocab))).astype(np.float32)
    params = [(1.0, 1.0, 0, 0.0), (1.0, 0.4, 0, 0.0), (1e-4, 0.9, 0, 0.0), (1.0, 1.0, 777, 0.0), (1e-4, 1.0, 0, 0.3), (1e-4, 0.9, 6000, 0.001),
              (1e-5, 1.0, 0, 0.0), (1.0, 0.9, 5000, 0.9999)]
    check(hip, logits, params, rng.random(8).astype(np.float32))


@pytest.mark.parametrize("vocab", [(1 << 17) - 1, 1 << 17, (1 << 17) + 1, (1 << 20) + 3, (1 << 24) - 1])
def test_counts_next_to_a_power_of_two(hip, rng, vocab):
    """Counts and weights share a word: all weights 1, and as many tokens as their bits hold."""
    logits = np.zeros((3, vocab), np.float32)
    logits[2] = rng.standard_normal(vocab)
    params = [(1.0, 1.0, 0, 0.0), (1.0, 0.75, vocab - 1, 0.0), (float("inf"), 1.0, vocab // 2 + 1, 0.0)]
    check(hip, logits, params, [0.9999, 0.6, 0.3])
