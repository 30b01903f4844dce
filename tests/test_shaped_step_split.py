"""How a mixed step with shaped scores shares the SMs between its two attention kernels, and that sharing them changes nothing."""
import numpy as np
import pytest
import torch

from nanopd_b200 import paged_forward


def context(chunks, positions, device="cpu", block=16):
    """``chunks``: (start, tokens).  Every sequence has pages of its own."""
    at, prefills, decodes = 0, [], []
    for start, n in chunks:
        pages = -(-(start + n) // block)
        prefills.append({"block_table": list(range(at, at + pages)), "start_position": start, "num_tokens": n})
        at += pages
    for p in positions:
        pages = p // block + 1
        decodes.append({"block_table": list(range(at, at + pages)), "position": p})
        at += pages
    ctx = {"num_prefill_tokens": sum(n for _, n in chunks), "num_decode_tokens": len(positions), "prefills": prefills, "decodes": decodes}
    return paged_forward.build_step_context(ctx, device), at


@pytest.mark.parametrize("window", [0, 1, 7, 64, 512, 513, 1000, 5000])
def test_visible_work(window):
    chunks, positions = [(0, 512), (100, 3), (700, 90), (510, 5), (0, 1)], [0, 6, 7, 63, 900, 8000]
    sc, _ = context(chunks, positions)
    w = window or 1 << 40
    pairs = sum(int(np.minimum(np.arange(s + 1, s + n + 1), w).sum()) for s, n in chunks)
    assert paged_forward._visible_work(sc, window) == (pairs, sum(min(p + 1, w) for p in positions))


def test_split_counts_what_a_window_leaves():
    """Contexts of 8000 tokens under a window of 1024 are contexts of 1024: the same share, or the same decision not to overlap."""
    split = lambda chunks, positions, **kw: paged_forward._sm_split(context(chunks, positions)[0], 32, 8, 128, 2, 148, **kw)  # noqa: E731
    for n in (4, 60, 128):
        assert split([(0, 1024)] * 4, [7999] * n, window=1024) == split([(0, 1024)] * 4, [1023] * n)
    assert split([(0, 1024)] * 4, [7999] * 4) is not None and split([(0, 1024)] * 4, [7999] * 4, window=1024) is None
    # queries far behind the window's length see a window each, no more
    pairs = paged_forward._visible_work(context([(4096, 512)], [3000])[0], 512)[0]
    assert pairs == 512 * 512


def test_split_gives_slower_scores_more():
    shares = [paged_forward._sm_split(context([(2048, 512)], [2200] * 128)[0], 32, 8, 128, 2, 148, shapings=s) for s in (0, 1, 2)]
    assert None not in shares and shares == sorted(shares) and shares[0] < shares[2]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [dict(score_cap=20.0), dict(window=300), dict(score_cap=20.0, window=1000, bias=True), dict(bias=True, window=40)])
def test_mixed_step_on_two_streams_equals_the_step_in_turn(kernels, monkeypatch, shape):
    monkeypatch.setattr(paged_forward, "_MIN_OVERLAP_SECONDS", 0.0)      # force the two-stream path at test size
    torch.manual_seed(3)
    dev, hq, hkv, d, dtype = "cuda:0", 8, 2, 128, torch.bfloat16
    sc, pages = context([(310, 150), (0, 90)], [700, 33, 1500, 64, 255, 1023, 12, 480], dev)
    total = sc.num_prefill_tokens + sc.num_decode_tokens
    k_cache, v_cache = (torch.randn(pages, hkv, 16, d, device=dev).to(dtype) for _ in range(2))
    q, k, v = (torch.randn(1, h, total, d, device=dev).to(dtype) for h in (hq, hkv, hkv))
    q *= 3
    kw = dict(score_cap=shape.get("score_cap", 0.0), window=shape.get("window", 0), distance_slopes=torch.rand(hq, device=dev) / 8 if "bias" in shape else None)
    assert paged_forward._sm_split(sc, hq, hkv, d, 2, 148, kw["window"], len([s for s in shape if s != "window"])) is not None
    outs = [paged_forward.paged_attention_step(sc, q, k, v, k_cache.clone(), v_cache.clone(), d ** -0.5, overlap=o, **kw)[0] for o in (False, True, True)]
    torch.cuda.synchronize()
    P = sc.num_prefill_tokens
    assert torch.equal(outs[0][:P], outs[1][:P])                         # prompt rows: the same kernel, the same tiles
    # decode rows: cut into other ranges; two roundings of the output and of the probabilities each
    assert (outs[0].float() - outs[1].float()).abs().max() <= 2 * (2 ** -8 + 2 ** -8) * float(v_cache.abs().max())
    assert torch.equal(outs[1], outs[2])
