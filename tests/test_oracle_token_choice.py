"""The token choice oracle: frequencies, the filters against brute force, special logits."""
import numpy as np
import pytest

from oracle.token_choice import choose, kept


def test_frequencies_follow_the_softmax():
    z = np.array([0.3, -1.0, 2.0, 0.0])
    got = np.bincount([choose(z, (i + 0.5) / 20000, 0.7)[0] for i in range(20000)], minlength=4) / 20000
    want = np.exp(z / 0.7) / np.exp(z / 0.7).sum()
    assert np.abs(got - want).max() <= 1 / 20000


@pytest.mark.parametrize("seed", range(4))
def test_filters_by_brute_force(seed):
    rng = np.random.default_rng(seed)
    z = np.round(rng.normal(size=12), 1)          # ties
    for k in (0, 1, 3, 12, 40):
        for p in (0.0, 0.3, 0.9, 1.0):
            for m in (0.0, 0.2, 1.0):
                w = np.exp((z - z.max()) / 0.9)
                ranks = [sum((z[j], -j) > (z[i], -i) for j in range(12)) for i in range(12)]
                in_k = [not k or r < k for r in ranks]
                total = sum(w[i] for i in range(12) if in_k[i])
                want = []
                for i in range(12):
                    above = sum(w[j] for j in range(12) if in_k[j] and z[j] > z[i])
                    stays = in_k[i] and (p >= 1 or above < p * total or z[i] == z.max()) and w[i] >= m
                    want.append(w[i] if stays else 0.0)
                assert np.allclose(kept(z, 0.9, k, p, m), want, rtol=1e-14)


def test_special_logits():
    assert choose([1.0, 3.0, 3.0, 2.0], 0.9, 0.0)[0] == 1                      # greedy, the lowest index
    assert choose([1.0, np.nan, 3.0], 0.99, 1e9)[0] == 2
    assert choose([np.nan, -np.inf], 0.5, 1.0)[0] == -1
    assert choose([np.inf, 0.0, np.inf], 0.4, 1.0)[0] == 0 and choose([np.inf, 0.0, np.inf], 0.6, 1.0)[0] == 2
    assert choose([1.0, 2.0, 9.0], 0.5, 1.0, allowed=np.array([True, True, False]))[0] == 1
    assert choose([0.0, 0.0], 0.5, 1.0)[0] == 1 and choose([0.0, 0.0], 1.0, 1.0)[0] == 1
    assert choose([0.0, 0.0, -np.inf], 2.0, 1.0)[0] == 1 and choose([0.0, 0.0], np.nan, 1.0)[0] == 0
