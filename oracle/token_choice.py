"""A token from logits and one uniform number, one row at a time, in float64 — test infrastructure only: the rule of
nanochat_amd/sampling.py's sample_tokens.

Pinned by tests/test_oracle_token_choice.py: softmax frequencies over evenly spaced uniform numbers, top-k, top-p and
min-p against brute force over subsets on small rows, the greedy choice, masks, infinities and NaN."""
import numpy as np


def weights(z, temperature):
    """exp((z - max) / T) over a row of allowed logits (-inf: not allowed); a +inf logit leaves only its equals."""
    top = z.max()
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        return np.where(z == top, 1.0, np.where(z == -np.inf, 0.0, np.exp(np.maximum((z - top) / temperature, -1e5))))


def kept(z, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """Weights (0: dropped) of a row of float64 logits, -inf where a token is not allowed."""
    n = z.size
    keep = z > -np.inf
    if 0 < top_k < n:
        order = np.lexsort((np.arange(n), -z))
        keep[order[top_k:]] = False
    w = np.where(keep, weights(z, temperature), 0.0)
    if top_p < 1:
        total = w.sum()
        values, which = np.unique(z, return_inverse=True)
        mass = np.bincount(which, w)
        above = mass[::-1].cumsum()[::-1] - mass
        # the largest value stays; above is exact where the sums are, and a border within their rounding is not tested
        keep &= (above < top_p * total)[which] | (z == z.max())
    keep &= w >= min(max(0.0 if np.isnan(min_p) else min_p, 0.0), 1.0)
    return np.where(keep, w, 0.0)


def choose(logits, uniform, temperature, top_k=0, top_p=1.0, min_p=0.0, allowed=None):
    """-> (token, margin): margin is how far the choice is from the next border, as a share of the weight."""
    z = np.asarray(logits, np.float64) + 0.0
    z = np.where(np.isnan(z), -np.inf, z)
    if allowed is not None:
        z = np.where(allowed, z, -np.inf)
    if not (z > -np.inf).any():
        return -1, 1.0
    if not temperature > 0:
        return int(np.argmax(z)), 1.0
    w = kept(z, float(temperature), int(top_k), float(top_p), float(min_p))
    share = w.cumsum()
    u = 0.0 if not uniform > 0 else float(uniform)
    if u >= 1:
        return int(np.flatnonzero(w)[-1]), 1.0
    target = u * share[-1]
    token = int(np.argmax(share > target))
    gaps = np.abs(share - target) / share[-1]
    return token, float(gaps.min()) if u > 0 else 1.0
