"""sampling.sample_tokens against the float64 oracle. The kernel's weights are off by at most 2^-47 of the largest each
(half a step of 2^-46), so a running share moves by less than vocab 2^-47, at most 2^-31 here: rows whose oracle choice is
nearer than 2^-30 to a border are not decided by it (a handful at most)."""
import numpy as np
import pytest
import torch

from nanochat_amd.sampling import sample_tokens
from oracle.token_choice import choose

pytestmark = pytest.mark.gpu
NEAR = 2.0 ** -30


def run(logits, device, uniform, temperature, top_k=None, top_p=None, min_p=None, mask=None, **kw):
    f = lambda x, d: None if x is None else torch.as_tensor(x).to(d).to(device)  # noqa: E731
    return sample_tokens(logits.to(device), f(uniform, torch.float32), f(temperature, torch.float32),
                         f(top_k, torch.int32), f(top_p, torch.float32), f(min_p, torch.float32),
                         None if mask is None else mask.to(device), **kw).cpu().numpy()


def compare(got, logits, uniform, temperature, top_k=None, top_p=None, min_p=None, allowed=None):
    z = logits.float().numpy()
    f32 = lambda x, r, d: d if x is None else float(np.float32(x[r]))  # noqa: E731
    skipped = 0
    for r in range(z.shape[0]):
        want, margin = choose(z[r], f32(uniform, r, 0), f32(temperature, r, 0), 0 if top_k is None else int(top_k[r]),
                              f32(top_p, r, 1.0), f32(min_p, r, 0.0), None if allowed is None else allowed[r])
        if margin < NEAR and want != got[r]:
            skipped += 1
            continue
        assert got[r] == want, (r, got[r], want, margin)
    assert skipped <= 1


def draws(rows, seed):
    rng = np.random.default_rng(seed)
    return (rng.random(rows).astype(np.float32), rng.uniform(0.3, 2.0, rows).astype(np.float32), rng)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 3, 64, 257, 4095, 4097, 32768, 50001, 65536, 70001])
def test_every_filter(device, vocab, dtype):
    rows = 24
    u, t, rng = draws(rows, vocab)
    t[::6] = 0.0
    logits = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32) * rng.choice([0.3, 2, 6], (rows, 1)))
    logits = logits.float().to(dtype)
    settings = dict(top_k=rng.choice([0, 1, 2, 40, vocab, vocab + 5, -3], rows),
                    top_p=rng.choice([1.0, 0.95, 0.5, 0.0, 1.5], rows), min_p=rng.choice([0.0, 0.0, 0.01, 1.0], rows))
    for names in ((), ("top_k",), ("top_p",), ("min_p",), ("top_k", "top_p", "min_p")):
        chosen = {n: settings[n] for n in names}
        compare(run(logits, device, u, t, **chosen), logits, u, t, **chosen)


@pytest.mark.parametrize("values", [1, 2, 7])
@pytest.mark.parametrize("vocab", [2000, 5000, 65536])
def test_ties(device, vocab, values):
    """Few distinct values: more equals in one range of values than the pairwise list holds; top-k cuts inside them."""
    rows = 16
    u, t, rng = draws(rows, values)
    logits = torch.from_numpy(rng.integers(0, values, (rows, vocab)).astype(np.float32) * 0.5 - 1.0)
    k = rng.integers(1, vocab, rows)
    compare(run(logits, device, u, t, top_k=k), logits, u, t, top_k=k)
    p = rng.random(rows).astype(np.float32)
    compare(run(logits, device, u, t, top_k=k, top_p=p), logits, u, t, top_k=k, top_p=p)


def test_crowded_ranges(device):
    """Thousands of distinct values within one of the 4,096 ranges, beside far outliers."""
    rows, vocab = 8, 40000
    u, t, rng = draws(rows, 5)
    z = (1.0 + rng.random((rows, vocab)) * 1e-3).astype(np.float32)
    z[:, 17], z[:, 30000] = -300.0, 3.0
    logits = torch.from_numpy(z)
    k = rng.integers(1, vocab, rows)
    p = rng.uniform(0.5, 0.999, rows).astype(np.float32)
    compare(run(logits, device, u, t, top_k=k), logits, u, t, top_k=k)
    compare(run(logits, device, u, t, top_p=p), logits, u, t, top_p=p)
    compare(run(logits, device, u, t, top_k=k, top_p=p), logits, u, t, top_k=k, top_p=p)


def test_masks(device):
    rows, vocab = 40, 1000
    u, t, rng = draws(rows, 6)
    logits = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32))
    words = rng.integers(0, 2 ** 32, (rows, 33), dtype=np.uint64).astype(np.uint32)     # a word more than needed
    words[0] = 0                                                                        # nothing allowed
    words[1] = 0
    words[1, 31] = 0xFFFFFF00                       # bits 8 .. 31 of the last word: token 1,000 and up, no token
    words[2] = 0
    words[2, 31] = 1 << 7                           # the last token alone
    bits = np.unpackbits(words.view(np.uint8).reshape(rows, -1), axis=1, bitorder="little")[:, :vocab].astype(bool)
    mask = torch.from_numpy(words.view(np.int32))
    t[3::4] = 0.0
    got = run(logits, device, u, t, mask=mask)
    compare(got, logits, u, t, allowed=bits)
    assert got[0] == got[1] == -1 and got[2] == vocab - 1
    k, p = np.full(rows, 30), np.full(rows, 0.8, np.float32)
    compare(run(logits, device, u, t, top_k=k, top_p=p, mask=mask), logits, u, t, top_k=k, top_p=p, allowed=bits)


def test_special_numbers(device):
    """Infinities, NaN, signed zeros, the type's lowest value; temperatures and uniform numbers outside their range."""
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    z = torch.tensor([
        [1.0, nan, 3.0, -inf, 0.0, -0.0], [nan, -inf, nan, -inf, nan, nan], [inf, 1.0, inf, nan, -inf, 0.0],
        [low, low, low, low, low, low], [0.0, -0.0, 0.0, -0.0, -1.0, low], [88.0, -88.0, 0.0, 1e38, -1e38, 1e-40],
        [low, 3e38, 0.0, 1.0, 2.0, 3.0]])
    rows = z.size(0)
    for u in (0.0, 0.4999, 0.9999999, 1.0, -1.0, nan, inf):
        for t in (1.0, 0.0, -1.0, nan, 1e-30, 1e30, inf, 0.5):
            uu, tt = np.full(rows, u, np.float32), np.full(rows, t, np.float32)
            got = run(z, device, uu, tt)
            want = [choose(z[r].numpy(), u, t)[0] for r in range(rows)]
            assert got.tolist() == want, (u, t)
            assert got[1] == -1
    for k, p, m in ((2, 1.0, 0.0), (0, 0.5, 0.0), (3, nan, nan), (0, -1.0, 2.0), (1, 0.0, 1.0)):
        uu, tt = np.full(rows, 0.7, np.float32), np.ones(rows, np.float32)
        got = run(z, device, uu, tt, np.full(rows, k), np.full(rows, p, np.float32), np.full(rows, m, np.float32))
        want = [choose(z[r].numpy(), 0.7, 1.0, k, p, m)[0] for r in range(rows)]
        assert got.tolist() == want, (k, p, m)


def test_strided_and_misaligned_rows(device):
    rows, vocab = 9, 1003
    u, t, rng = draws(rows, 7)
    for dtype in (torch.float32, torch.bfloat16):
        full = torch.from_numpy(rng.normal(size=(rows, 1030)).astype(np.float32)).to(dtype)
        for first in (0, 1, 2, 8):
            view = full.to(device)[:, first:first + vocab]
            got = sample_tokens(view, torch.from_numpy(u).to(device), torch.from_numpy(t).to(device)).cpu().numpy()
            compare(got, full[:, first:first + vocab], u, t)


def test_frequencies(device):
    """20,000 evenly spaced uniform numbers over one row: every token as often as its share, to one draw."""
    rng = np.random.default_rng(8)
    z = torch.from_numpy(rng.normal(size=300).astype(np.float32) * 2)
    n = 20000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = run(z.expand(n, -1).contiguous(), device, u, np.full(n, 0.9, np.float32))
    w = np.exp(z.double().numpy() / np.float32(0.9).astype(np.float64))
    # a border takes or loses at most the draw at it, and u itself is rounded by up to 2^-25
    assert np.abs(np.bincount(got, minlength=300) - n * w / w.sum()).max() <= 2.01


def test_rows_do_not_depend_on_each_other_and_repeat(device):
    rows, vocab = 64, 5000
    u, t, rng = draws(rows, 9)
    logits = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32))
    k, p = rng.integers(0, 50, rows), rng.uniform(0.5, 1.1, rows).astype(np.float32)
    all_rows = run(logits, device, u, t, top_k=k, top_p=p)
    assert np.array_equal(all_rows, run(logits, device, u, t, top_k=k, top_p=p))
    for r in (0, 31, 63):
        s = slice(r, r + 1)
        assert run(logits[s], device, u[s], t[s], top_k=k[s], top_p=p[s])[0] == all_rows[r]


def test_captured(device):
    """One graph, replayed with new logits and numbers, eager calls between the replays."""
    rows, vocab = 12, 3000
    rng = np.random.default_rng(10)
    logits = torch.zeros(rows, vocab, device=device)
    u, t = torch.zeros(rows, device=device), torch.ones(rows, device=device)
    p = torch.full((rows,), 0.9, device=device)
    out = torch.empty(rows, dtype=torch.int32, device=device)
    sample_tokens(logits, u, t, top_p=p, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample_tokens(logits, u, t, top_p=p, out=out)
    for _ in range(4):
        logits.copy_(torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32)))
        u.copy_(torch.from_numpy(rng.random(rows).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        eager = sample_tokens(logits, u, t, top_p=p)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_refusals(device):
    z, u = torch.zeros(3, 8, device=device), torch.zeros(3, device=device)
    sample_tokens(z, u, u)
    for bad in (dict(logits=z[0]), dict(logits=z.cpu()), dict(uniform=u[:2]), dict(temperature=u.cpu()), dict(logits=z.t()),
                dict(logits=z[:1].expand(3, 8)), dict(logits=z[:, :0]), dict(mask=torch.zeros(3, 0, dtype=torch.int32, device=device)),
                dict(mask=torch.zeros(2, 1, dtype=torch.int32, device=device)), dict(out=torch.zeros(4, dtype=torch.int32, device=device))):
        with pytest.raises(ValueError):
            sample_tokens(**{**dict(logits=z, uniform=u, temperature=u), **bad})
    for bad in (dict(logits=z.half()), dict(uniform=u.double()), dict(top_k=u), dict(top_p=u.int()),
                dict(mask=torch.zeros(3, 1, dtype=torch.int64, device=device)), dict(out=u)):
        with pytest.raises(TypeError):
            sample_tokens(**{**dict(logits=z, uniform=u, temperature=u), **bad})
    assert sample_tokens(z[:0], u[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("vocab", [700, 8192, 8193, 20000, 262144, 262145])
def test_few_allowed_tokens(device, vocab):
    """Fewer allowed tokens than top-k asks for, in few places of the row or crowded in one, and none at all."""
    rows = 10
    u, t, rng = draws(rows, 11)
    logits = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32))
    bits = np.zeros((rows, -(-vocab // 32) * 32), bool)
    for r in range(rows):
        if r % 3 == 0:
            bits[r, rng.integers(0, vocab, r)] = True
        elif r % 3 == 1:
            at = int(rng.integers(0, vocab - 200))
            bits[r, at:at + 40 * r] = True
        else:
            bits[r, vocab - r:vocab] = True
    bits[:, vocab:] = False
    mask = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32))
    allowed = bits[:, :vocab]
    for k in (1, 2, 50, 128, 129, 400):
        for p in (1.0, 0.9):
            kk, pp = np.full(rows, k), np.full(rows, p, np.float32)
            compare(run(logits, device, u, t, top_k=kk, top_p=pp, mask=mask), logits, u, t, top_k=kk, top_p=pp, allowed=allowed)
    compare(run(logits, device, u, t, top_p=np.full(rows, 0.7, np.float32), mask=mask), logits, u, t,
            top_p=np.full(rows, 0.7, np.float32), allowed=allowed)


@pytest.mark.parametrize("order", ["up", "down", "blocks"])
def test_sorted_rows(device, order):
    """Logits in an order that puts the largest into few threads, and equal logits everywhere."""
    rows, vocab = 8, 30000
    u, t, rng = draws(rows, 12)
    z = np.sort(rng.normal(size=(rows, vocab)).astype(np.float32), axis=1)
    if order == "down":
        z = z[:, ::-1].copy()
    elif order == "blocks":
        z = np.roll(z.reshape(rows, -1, 8)[:, rng.permutation(vocab // 8)].reshape(rows, vocab), 3, axis=1)
        z[4:] = 1.5
    logits = torch.from_numpy(z)
    for k in (1, 3, 100, 127, 128, 129, 5000):
        kk = np.full(rows, k)
        compare(run(logits, device, u, t, top_k=kk), logits, u, t, top_k=kk)
    pp = rng.uniform(0.1, 1.0, rows).astype(np.float32)
    compare(run(logits, device, u, t, top_p=pp), logits, u, t, top_p=pp)


def test_calls_of_many_and_few_rows(device):
    """More rows than are cut into slices, and a call of few between them on the same workspace."""
    vocab, rows = 9000, 1500
    u, t, rng = draws(rows, 13)
    logits = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32) * 3)
    k = np.where(rng.random(rows) < 0.5, 0, 30)
    p = np.full(rows, 0.9, np.float32)
    got = run(logits, device, u, t, top_k=k, top_p=p)
    few = run(logits[:3], device, u[:3], t[:3], top_k=k[:3], top_p=p[:3])
    assert np.array_equal(few, got[:3]) and np.array_equal(got, run(logits, device, u, t, top_k=k, top_p=p))
    some = rng.permutation(rows)[:60]
    compare(got[some], logits[some], u[some], t[some], top_k=k[some], top_p=p[some])


@pytest.mark.parametrize("rows,vocab,with_k", [(70, 65536, True), (260, 20000, False), (40, 65536, False), (2100, 9000, True),
                                               (3, 262144, False), (2, 300001, True)])
def test_many_rows(device, rows, vocab, with_k):
    """Batches on either side of where rows stop being cut into slices, each row with settings of its own."""
    u, t, rng = draws(rows, rows)
    t[::5] = 0.0
    logits = torch.from_numpy((rng.normal(size=(rows, vocab)) * rng.choice([0.5, 2.5], (rows, 1))).astype(np.float32))
    k = rng.choice([0, 1, 2, 50, 128, 129, 1000], rows) if with_k else None
    p = rng.choice([1.0, 0.95, 0.3], rows).astype(np.float32)
    m = rng.choice([0.0, 0.02], rows).astype(np.float32)
    got = run(logits, device, u, t, top_k=k, top_p=p, min_p=m)
    some = rng.permutation(rows)[:48]
    compare(got[some], logits[some], u[some], t[some], top_k=None if k is None else k[some], top_p=p[some], min_p=m[some])


@pytest.mark.parametrize("rows", [5, 80, 260])
@pytest.mark.parametrize("period,run_of", [(256, 16), (2048, 256), (4096, 64)])
def test_top_tokens_crowded_in_few_threads(device, rows, period, run_of):
    """A top-k whose candidates may outnumber their list: the largest tokens in runs that few threads read."""
    vocab = 65536
    u, t, rng = draws(rows, 14)
    z = rng.normal(size=(rows, vocab)).astype(np.float32)
    z.reshape(rows, -1, period)[:, :, :run_of] += 20
    z[1] = 2.0                                                       # equals everywhere
    logits = torch.from_numpy(z)
    k = rng.choice([2, 100, 128], rows)
    got = run(logits, device, u, t, top_k=k)
    some = rng.permutation(rows)[:20]
    some[0] = 1
    compare(got[some], logits[some], u[some], t[some], top_k=k[some])


def test_one_row_of_odd_width(device):
    """A single row's stride is no one's business: aligned loads, and a last slice that ends inside a group of four."""
    for vocab in (8193, 50257, 50258, 300003):
        u, t, rng = draws(1, vocab)
        for dtype in (torch.float32, torch.bfloat16):
            logits = torch.from_numpy(rng.normal(size=(1, vocab)).astype(np.float32) * 2).to(dtype)
            for k, p in ((0, 0.9), (40, 0.9), (0, 1.0)):
                kk, pp = np.full(1, k), np.full(1, p, np.float32)
                compare(run(logits, device, u, t, top_k=kk, top_p=pp), logits, u, t, top_k=kk, top_p=pp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(4, 20000), (200, 20000), (300, 20001)])
def test_extremes_and_masks_in_every_form(device, rows, vocab, dtype):
    """Rows in slices, a row a workgroup, two workgroups a CU: NaN and infinities in allowed and masked places, the type's
    lowest and largest values beside ordinary ones (a range of values past the largest number), masks that leave one token."""
    u, t, rng = draws(rows, 15)
    t[::7] = 0.0
    z = rng.normal(size=(rows, vocab)).astype(np.float32)
    big = torch.finfo(dtype).max
    for r in range(rows):
        at = rng.integers(0, vocab, 40)
        z[r, at] = rng.choice([np.nan, -np.inf, -big, 0.0, -0.0], 40)
        if r % 4 == 1:
            z[r, at[0]] = big
        elif r % 4 == 2:
            z[r, at[:3]] = np.inf
        elif r % 4 == 3:
            z[r] = np.where(rng.random(vocab) < 0.5, -big, z[r])
    logits = torch.from_numpy(z).to(dtype)
    bits = rng.random((rows, -(-vocab // 32) * 32)) < 0.6
    bits[::5] = False
    bits[::5, 777] = True
    bits[5::10, 777] = False
    mask = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32))
    k, p = rng.choice([0, 1, 60, 3000], rows), rng.choice([1.0, 0.9], rows).astype(np.float32)
    m = rng.choice([0.0, 0.1], rows).astype(np.float32)
    some = rng.permutation(rows)[:40]
    some[:3] = [0, min(5, rows - 1), 1]
    for allowed, words in ((None, None), (bits[:, :vocab], mask)):
        got = run(logits, device, u, t, top_k=k, top_p=p, min_p=m, mask=words)
        compare(got[some], logits[some], u[some], t[some], top_k=k[some], top_p=p[some], min_p=m[some],
                allowed=None if allowed is None else allowed[some])
