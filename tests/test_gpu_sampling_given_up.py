"""Rows that the workgroups sharing them give up because the others do not come (their patience set to next to nothing from the
host, so that most rows end this way) get the tokens that they get otherwise, and leave the workspace as it was."""
import numpy as np
import pytest
import torch

from nanochat_amd.native import check, hip_library, pointer, stream
from nanochat_amd.sampling import sample_tokens, sample_workspace_bytes

pytestmark = pytest.mark.gpu
COUNTS = (2 * 8 + 256) * 128   # a 128-byte line for each queue's two counts and each row


def impatient(logits, u, t, k, p, m, mask, workspace, patience):
    rows, vocab = logits.shape
    out = torch.full((rows,), -7, dtype=torch.int32, device=logits.device)
    check(hip_library().nc_debug_sample_tokens(
        pointer(logits), logits.dtype == torch.bfloat16, vocab, rows, vocab, pointer(u), pointer(t), pointer(k), pointer(p),
        pointer(m), pointer(mask) if mask is not None else None, mask.size(1) if mask is not None else 0, pointer(out),
        pointer(workspace), workspace.numel(), patience, stream()))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 8193), (3, 20001), (16, 65536), (40, 70001), (16, 262144), (2, 140000)])
def test_given_up_rows(device, rows, vocab, dtype):
    rng = np.random.default_rng(rows + vocab)
    on = lambda x, d: torch.as_tensor(x).to(d).to(device)  # noqa: E731
    z = rng.normal(size=(rows, vocab)).astype(np.float32) * rng.choice([0.3, 2.5], (rows, 1))
    if rows > 2:
        z[2] = 1.5                                                   # equals everywhere
    logits = on(z, dtype)
    u, t = on(rng.random(rows), torch.float32), on(np.where(rng.random(rows) < 0.2, 0.0, rng.uniform(0.4, 2.0, rows)), torch.float32)
    bits = rng.random((rows, -(-vocab // 32) * 32)) < 0.7
    bits[rows // 2] = False                                          # nothing allowed
    words = on(np.packbits(bits, axis=1, bitorder="little").view(np.int32), torch.int32)
    workspace = torch.zeros(sample_workspace_bytes(rows, vocab), dtype=torch.uint8, device=device)
    for mask in (None, words):
        for ks, ps, ms in (([0], [1.0], [0.0]), ([0], [0.9, 0.3], [0.0, 0.01]), ([129, 4000, vocab], [1.0, 0.95], [0.0]),
                           ([0, 1, 40, 128, 129, 4000], [1.0, 0.9], [0.0, 0.05])):
            k, p, m = (on(rng.choice(x, rows), d) for x, d in ((ks, torch.int32), (ps, torch.float32), (ms, torch.float32)))
            want = sample_tokens(logits, u, t, k, p, m, mask)
            for patience in (0, 1, 4):
                got = impatient(logits, u, t, k, p, m, mask, workspace, patience)
                assert torch.equal(got, want), (patience, got, want)
                assert not bool(workspace[:COUNTS].any())
    if rows > 1:
        assert int(want[rows // 2]) == -1


def test_four_streams_at_once(device):
    """More rows in slices than the device runs at once, from four streams: every call ends, with its own tokens."""
    rows, vocab = 16, 140000
    rng = np.random.default_rng(1)
    logits = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32)).to(device)
    u = torch.from_numpy(rng.random((4, rows)).astype(np.float32)).to(device)
    t, p = torch.ones(rows, device=device), torch.full((rows,), 0.9, device=device)
    want = [sample_tokens(logits, u[i], t, top_p=p) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [[] for _ in streams]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(sample_tokens(logits, u[i], t, top_p=p))
    torch.cuda.synchronize()
    for i in range(4):
        for tokens in got[i]:
            assert torch.equal(tokens, want[i])


def test_patience_is_checked(device):
    z, u = torch.zeros(1, 8, device=device), torch.zeros(1, device=device)
    i, ws = torch.zeros(1, dtype=torch.int32, device=device), torch.zeros(16, dtype=torch.uint8, device=device)
    for patience in (-1, 65537):
        assert hip_library().nc_debug_sample_tokens(pointer(z), 0, 8, 1, 8, pointer(u), pointer(u), None, None, None, None, 0,
                                                    pointer(i), pointer(ws), 16, patience, stream()) == -2
