"""GPU: caps of any size beside the scores, decode and prompts, against a plain form in 64 bits."""
import pytest
import torch

import test_gpu_scored_attention as decode
import test_gpu_scored_prefill as prompt
from oracle import shaped_oracle

pytestmark = pytest.mark.gpu

CAPS = [200.0, 1e3, 1e5, 1e6, 1e7, 1e9, 1e20, 1e38]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("hq,hkv,d", [(12, 2, 128), (16, 16, 64), (8, 2, 256)])
def test_large_caps_in_decode(kernels, hq, hkv, d, cap):
    """Scores of up to 15 or so under a cap that leaves them as they are: the rows are those of that cap, whatever its size."""
    lens = [1, 16, 100, 700, 333]
    q, kc, vc, bt, sl, scale = decode.make(lens, hq, hkv, d, 16, torch.float16, gain=3.0)
    decode.check(kernels, q, kc, vc, bt, sl, scale, cap)
    decode.check(kernels, q, kc, vc, bt, sl, scale, cap, decode.slopes_for(hq), 60)
    decode.check(kernels, q, kc, vc, bt, sl, scale, cap, max_ctas=140)


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("hq,hkv,d", [(12, 2, 128), (16, 16, 64), (8, 2, 256)])
def test_large_caps_in_prompts(kernels, hq, hkv, d, cap):
    chunks = [(0, 200), (70, 300)]
    q, kc, vc, bt = prompt.make(chunks, hq, hkv, d, 16, torch.float16, gain=3.0)
    prompt.check(kernels, q, kc, vc, bt, chunks, cap)
    prompt.check(kernels, q, kc, vc, bt, chunks, cap, prompt.slopes_for(hq), 90)


@pytest.mark.parametrize("cap", [c for c in CAPS if c >= 1e5])
def test_a_large_cap_changes_nothing_that_the_scores_show(kernels, cap):
    """A cap a thousand times the largest score and more moves a score by less than 1e-6 of it; the plain form of the same
    operator is that close.  (Probabilities move by 2^-11 or less in fp16, and by 15 * 1.2e-6 through the score.)"""
    chunks = [(0, 250)]
    q, kc, vc, bt = prompt.make(chunks, 12, 2, 128, 16, torch.float16, gain=3.0)
    out, plain = torch.empty_like(q), torch.empty_like(q)
    prompt.call(kernels, out, q, kc, vc, bt, chunks, 128 ** -0.5, score_cap=cap)
    prompt.call(kernels, plain, q, kc, vc, bt, chunks, 128 ** -0.5)
    assert (out.float() - plain.float()).abs().max() <= 2 ** -8


@pytest.mark.parametrize("cap,gain", [(800.0, 60.0), (800.0, 200.0), (30.0, 8.0), (30.0, 12.0), (50.0, 40.0), (5000.0, 400.0)])
@pytest.mark.parametrize("bias,window", [(False, 0), (True, 0), (False, 70)])
def test_scores_around_large_caps(kernels, cap, gain, bias, window):
    """Scores that reach the cap.  Beside the bound that scores of up to 60 have, the score itself is off by a share of its
    size: 2.2e-6 (the prompt kernel's shorter polynomial), 5e-7 (the sums of 128 products) and 2.4e-7 (roundings of the product
    with the scale and of the exponent's difference); all of it moves a row by at most twice that times A."""
    chunks = [(0, 200), (90, 150)]
    q, kc, vc, bt = prompt.make(chunks, 12, 2, 128, 16, torch.bfloat16, gain=gain)
    slopes = prompt.slopes_for(12) if bias else None
    scale, at = 128 ** -0.5, 0
    out = torch.full_like(q, float("nan"))
    prompt.call(kernels, out, q, kc, vc, bt, chunks, scale, score_cap=cap, distance_slopes=slopes, window=window)
    S = min(cap, 7 * gain)                                  # no score of a deviation of `gain` is beyond seven of it, or the cap
    for c, (start, n) in enumerate(chunks):
        want, A, l = shaped_oracle.attend(q[at:at + n], kc, vc, bt[c], start, scale, cap, slopes, window)
        tol = shaped_oracle.attention_tolerance(want, A, l, start + n, q.dtype, float(vc.abs().max())) + 2 * A * S * 3e-6
        off = (out[at:at + n].double() - want).abs()
        assert (off <= tol).all(), f"chunk {c}: worst {float((off / tol).max()):.2f} of the tolerance"
        # the last token of the chunk as a decode step
        one = torch.empty_like(q[:1])
        kernels.paged_scored_attention(one, q[at + n - 1:at + n], kc, vc, bt[c:c + 1], torch.tensor([start + n], dtype=torch.int32, device="cuda"),
                                       scale, 16, bt.size(1), score_cap=cap, distance_slopes=slopes, window=window)
        assert ((one[0].double() - want[-1]).abs() <= tol[-1]).all()
        at += n


@pytest.mark.parametrize("cap", [1.1e38, 3e38, 1e-31])
def test_caps_that_are_refused(kernels, cap):
    q, kc, vc, bt, sl, scale = decode.make([5], 12, 2, 128, 16, torch.float16)
    with pytest.raises(RuntimeError, match="cap"):
        kernels.paged_scored_attention(torch.empty_like(q), q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=cap)
