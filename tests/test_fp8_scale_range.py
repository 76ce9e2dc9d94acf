"""The scales that the 8-bit products fetch, on the host. Their kernels fetch stages of 128 columns ahead, up to two past the
last, and with every fourth stage a dword of scales for each row. What lies past a buffer's range is not read, so the range has to
end where a scale tensor may: fp8_linear accepts any view whose last row is there up to its scales' padding to a dword, as the last
columns of wider rows are."""
import re
import subprocess
from pathlib import Path

import pytest
import torch

from nanochat_amd import fp8_linear as fl, native

AHEAD = 2   # stages past the last


@pytest.fixture(scope="module")
def scale_range(tmp_path_factory):
    exe = tmp_path_factory.mktemp("range") / "range"
    source = Path(__file__).parent / "fp8_scale_range.hip"
    subprocess.run([native.hipcc(), "--offload-host-only", "-O1", "-std=c++17", f"-I{native.CSRC}", f"-I{native.INCLUDE}", "-o",
                    str(exe), str(source)], check=True, capture_output=True)
    return lambda *args: int(subprocess.run([str(exe), *map(str, args)], check=True, capture_output=True, text=True).stdout)


def views(rows, blocks, pitch):
    """Scales [rows, blocks] at a pitch: the last columns of wider rows, at the very end of their storage."""
    whole = torch.zeros(rows, pitch, dtype=torch.uint8).view(fl.SCALE)
    return whole[:, pitch - -(-blocks // 4) * 4:][:, :blocks]


@pytest.mark.parametrize("blocks", [1, 3, 4, 8, 13, 16, 52])
@pytest.mark.parametrize("rows,wider", [(1, 0), (1, 12), (8, 0), (8, 48), (256, 4), (300, 20)])
def test_no_scale_is_read_past_the_end_of_its_tensor(scale_range, monkeypatch, rows, wider, blocks):
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    pitch = -(-blocks // 4) * 4 + wider
    scale = views(rows, blocks, pitch)
    assert fl._check_scale(scale, "scale", rows, blocks * 128, scale.device) == pitch
    there = scale.untyped_storage().nbytes() - scale.storage_offset()
    for first in range(0, rows, 256):                        # a tile's rows
        count = min(256, rows - first)
        end = scale_range(count, pitch, blocks)
        for row in range(256):
            for j in range(0, blocks + AHEAD + 1, 4):
                at = row * pitch + j
                read = at < end
                assert not read or first * pitch + at + 4 <= there, (row, j)
                assert read or row >= count or j >= blocks, (row, j)   # and none that counts is left out


def test_every_scale_buffer_has_that_range():
    made = []
    for name in ("fp8_gemm.hip", "fp8_grad.hip", "fp8_skinny.hip"):
        for line in (native.CSRC / name).read_text().splitlines():
            if re.search(r"f8_(words|rsrc)\([^;]*\b(as|ws|xs)\b[^;]*;", line):
                made.append(line)
    assert len(made) >= 5 and all("f8_scale_range(" in line for line in made)
