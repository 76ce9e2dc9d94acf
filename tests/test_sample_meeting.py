"""The token choice's waits between workgroups (nanochat_amd/csrc/nc_meeting.h), replayed on the host: a workgroup that
waits holds a place on a CU that the ones it waits for may need, so with waits that have no bound several launches at once,
or one on a device of few CUs, can stop for good. With the kernel's bounded waits every launch ends, each row is chosen
once, and the counts are zero again."""
import subprocess
from pathlib import Path

import pytest

from nanochat_amd import native


@pytest.fixture(scope="module")
def replay(tmp_path_factory):
    exe = tmp_path_factory.mktemp("replay") / "replay"
    source = Path(__file__).parent / "sample_meeting_replay.hip"
    subprocess.run([native.hipcc(), "--offload-host-only", "-O2", "-std=c++17", f"-I{native.CSRC}", "-o", str(exe), str(source)],
                   check=True, capture_output=True)

    def run(*args):
        return subprocess.run([str(exe), *map(str, args)], check=True, capture_output=True, text=True, timeout=120).stdout.strip()

    return run


# launches, XCDs, places an XCD, rows, workgroups a row: what runs at once on 256 CUs, on one XCD of 32, on a few CUs
CROWDED = [(3, 8, 64, 16, 32), (4, 8, 64, 24, 17), (1, 1, 64, 16, 32), (2, 1, 64, 8, 20), (1, 1, 16, 3, 32), (8, 8, 64, 16, 32),
           (1, 1, 1, 2, 2)]


@pytest.mark.parametrize("sizes", CROWDED)
def test_waits_without_bound_can_stop_for_good(replay, sizes):
    """What the replay is able to show: the same tickets and words with waits that have no bound."""
    assert "stuck" in {replay(*sizes, 3, -1, seed) for seed in range(3)}


@pytest.mark.parametrize("patience", [0, 1, 7, 60])
@pytest.mark.parametrize("sizes", CROWDED + [(1, 8, 64, 16, 32), (1, 8, 64, 1, 8), (2, 8, 64, 51, 10)])
def test_every_launch_ends(replay, sizes, patience):
    for seed in range(4):
        assert replay(*sizes, 1 + seed * 2, patience, seed) == "ended", seed
