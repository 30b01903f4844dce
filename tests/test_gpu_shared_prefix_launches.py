"""GPU: the plan, prefix and tail launches of the shared-prefix operator, on batches that the operator would answer in one
launch if the number of CTAs were not limited."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_an_odd_number_of_stages_of_a_cta(kernels):
    """Five warps of one stage each leave the barriers' end in the middle of a 16-byte piece."""
    here = Path(__file__).resolve()
    env = dict(os.environ, NPD_DECODE_WARPS="5", NPD_DECODE_STAGES="1")
    res = subprocess.run([sys.executable, "-m", "pytest", str(here.with_name("test_gpu_shared_prefix.py")), "-q", "-x", "-p", "no:cacheprovider",
                          "-k", "test_shapes"], env=env, capture_output=True, text=True, timeout=600, cwd=str(here.parents[1]))
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-2000:]
