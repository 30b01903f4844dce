"""CPU: where the tail kernel of the shared-prefix operator keeps the rows it joins, restated from its source."""
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parents[1] / "nanopd_b200" / "csrc" / "decode_kernel.cuh").read_text()


def test_the_source_is_what_is_restated_here():
    assert "const size_t bar_bytes = MODE == kTail ? ((size_t)nwarps * nst * 8 + 15) / 16 * 16" in SOURCE
    assert "reinterpret_cast<int *>(sbase + (size_t)nwarps * nst * STAGE_BYTES + bar_bytes)" in SOURCE
    assert re.search(r"scratch = reinterpret_cast<float \*>\(pre \+ \(p\.num_seqs \+ 4\) / 4 \* 4\) \+ warp \* \(\(joined_floats\(D, p\.group\) \+ 3\) / 4 \* 4\);", SOURCE)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_scratch_is_aligned_and_inside_the_cta(d):
    """Every warp's rows lie on a 16-byte boundary (read as float4), behind the prefix and within what the launcher asks for,
    for every number of warps and stages that the tuning knobs allow."""
    for warps in range(1, 13):
        for stages in range(1, 5):
            for seqs in (1, 2, 3, 4, 5, 133, 4096):
                for group in (1, 3, 7, 8, 16):
                    joined = (group * (d + 4) + 2 * group + 3) // 4 * 4
                    bars = (warps * stages * 8 + 15) // 16 * 16
                    pre = warps * stages * 64 * d + bars
                    scratch = pre + (seqs + 4) // 4 * 16
                    assert scratch % 16 == 0 and joined * 4 % 16 == 0 and scratch >= pre + 4 * (seqs + 1)
                    asked = 1024 + warps * stages * (64 * d + 8) + (seqs + 1) * 4 + 32 + warps * joined * 4
                    assert scratch + warps * joined * 4 <= asked - 1008        # the ring's alignment takes up to 1008 bytes
