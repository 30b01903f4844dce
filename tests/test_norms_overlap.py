"""Outputs of the norms between blocks that cover a weight: refused, by addresses on the CPU and by the operator on the GPU."""
import pytest
import torch

from nanopd_b200 import norms


def clear_of(w, out, stride, rows=4, row=64):
    extent = (rows - 1) * stride + row
    far = 1 << 20
    return norms._clear_of(w, out, extent, stride, far, extent, stride, row) and norms._clear_of(w, far, extent, stride, out, extent, stride, row)


def test_addresses():
    assert clear_of(0, 64, 64) and clear_of(64 + 256, 64, 64)                    # in front, behind
    assert not clear_of(0, 63, 64) and not clear_of(64 + 255, 64, 64) and not clear_of(128, 64, 64)
    assert clear_of(64, 0, 192) and clear_of(128, 0, 192) and clear_of(192 + 96, 0, 192)      # between the rows
    assert not clear_of(32, 0, 192) and not clear_of(160, 0, 192) and not clear_of(192, 0, 192)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["weight", "post_weight", "gate"])
@pytest.mark.parametrize("output", ["residual_out", "out"])
def test_outputs_that_cover_a_weight_are_refused(which, output):
    dev, bf16 = "cuda:0", torch.bfloat16
    x, r, w = torch.randn(4, 256, device=dev).to(bf16), torch.randn(4, 256, device=dev).to(bf16), torch.ones(256, device=dev, dtype=bf16)
    buf = torch.ones(6, 512, device=dev, dtype=bf16)
    want = norms.residual_norms(x, r, w, post_weight=w, gate=w)
    for covered in (buf[2, :256], buf[2, 8:264], buf[4, :256], buf[5, 248:504]):
        with pytest.raises(RuntimeError, match="overlaps"):
            norms.residual_norms(x, r, **{**dict(weight=w, post_weight=w, gate=w), which: covered}, **{output: buf[2:, :256]})
    buf.fill_(1)
    free = (buf[1, 256:], buf[0, :256]) if which == "gate" else (buf[1, 256:], buf[0, :256], buf[3, 256:])
    for beside in free:
        got = norms.residual_norms(x, r, **{**dict(weight=w, post_weight=w, gate=w), which: beside}, **{output: buf[2:, :256]})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
