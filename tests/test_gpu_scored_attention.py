"""GPU: paged decode attention with shaped scores (cap, distance bias, window) against a plain form in 64 bits."""
import pytest
import torch

from nanopd_b200 import workloads
from oracle import shaped_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(lens, hq, hkv, d, block, dtype, seed=0, gain=1.0):
    b = workloads.make_decode_batch([max(0, n - 1) for n in lens], hq, hkv, d, block, dtype, device=DEV, seed=seed)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return b.query * gain, b.k_cache, b.v_cache, b.block_tables, sl, b.scale


def poison(kc, vc, bt, lens, window, value=float("nan")):
    """Everything that a row may not see: slots behind a sequence and before its window, and table entries of pages wholly
    before it."""
    block = kc.size(2)
    seen = torch.zeros(kc.size(0), block, dtype=torch.bool)
    bt_cpu = bt.cpu()
    for s, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        for j in range(lo, n):
            seen[int(bt_cpu[s, j // block]), j % block] = True
        bt_cpu[s, :lo // block] = -7
    hide = (~seen).to(kc.device)
    kc.permute(0, 2, 1, 3)[hide] = value
    vc.permute(0, 2, 1, 3)[hide] = value
    bt.copy_(bt_cpu)


def slopes_for(hq):
    return torch.exp2(-8.0 * torch.arange(1, hq + 1, dtype=torch.float32, device=DEV) / hq)


def check(kernels, q, kc, vc, bt, sl, scale, cap=0.0, slopes=None, window=0, max_ctas=0, rows=None):
    out = torch.full_like(q, float("nan"))
    kernels.paged_scored_attention(out, q, kc, vc, bt, sl, scale, kc.size(2), bt.size(1), score_cap=cap, distance_slopes=slopes,
                                   window=window, max_ctas=max_ctas)
    torch.cuda.synchronize()
    want, A, l = shaped_oracle.attend_single(q, kc, vc, bt, sl, scale, cap, slopes, window)
    v_max = float(vc[torch.isfinite(vc)].abs().max())
    tol = shaped_oracle.attention_tolerance(want, A, l, int(sl.max()), q.dtype, v_max)
    off = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (off <= tol).all(), f"worst {float((off / tol).max()):.2f} of the tolerance"
    return out


SHAPES = [
    (12, 2, 128, 16, [16, 100, 512, 333, 1, 47, 250, 64]),
    (32, 8, 128, 16, [1, 2, 15, 16, 17, 31, 33, 900]),
    (40, 2, 128, 16, [5, 700, 33]),                 # group 20: two virtual kv heads per head
    (16, 16, 64, 8, [9, 130, 77, 1500]),
    (14, 2, 64, 32, [31, 32, 33, 640]),
    (8, 2, 256, 32, [31, 32, 33, 1000, 7]),
    (24, 8, 128, 4, [3, 4, 5, 257]),
    (16, 1, 256, 16, [1, 300]),                     # group 16 at head size 256: two virtual kv heads
]
SCORES = [(50.0, False, 0), (0.0, True, 0), (0.0, False, 40), (30.0, True, 33), (20.0, False, 1), (0.0, True, 16), (5.0, True, 100000)]


@pytest.mark.parametrize("cap,bias,window", SCORES)
@pytest.mark.parametrize("hq,hkv,d,block,lens", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_shapes_and_scores(kernels, dtype, hq, hkv, d, block, lens, cap, bias, window):
    q, kc, vc, bt, sl, scale = make(lens, hq, hkv, d, block, dtype, gain=3.0 if cap else 1.0)
    poison(kc, vc, bt, lens, window)
    slopes = slopes_for(hq) if bias else None
    check(kernels, q, kc, vc, bt, sl, scale, cap, slopes, window)                  # the small-batch form where it applies
    check(kernels, q, kc, vc, bt, sl, scale, cap, slopes, window, max_ctas=100)    # the streaming form


@pytest.mark.parametrize("window", [1, 15, 16, 17, 128, 4096])
def test_windows_over_long_contexts(kernels, window):
    lens = [4097, 4096, 4095, 1, 9000, 16, 0, 2500]
    q, kc, vc, bt, sl, scale = make(lens, 32, 8, 128, 16, torch.bfloat16, gain=2.0)
    poison(kc, vc, bt, lens, window)
    out = check(kernels, q, kc, vc, bt, sl, scale, 50.0, None, window)
    assert (out[6] == 0).all()


def test_empty_batch_and_empty_sequences(kernels):
    q, kc, vc, bt, sl, scale = make([0, 5, 0], 12, 2, 128, 16, torch.float16)
    for cap in (0, 100):
        out = check(kernels, q, kc, vc, bt, sl, scale, 30.0, None, 3, max_ctas=cap)
        assert (out[0] == 0).all() and (out[2] == 0).all()
    kernels.paged_scored_attention(q[:0], q[:0], kc, vc, bt[:0], sl[:0], scale, 16, bt.size(1), score_cap=30.0)


def test_without_shaping_agrees_with_the_plain_operator(kernels):
    """Cap 0, no slopes, no window: the same scores.  The two split a sequence at other places, so their sums differ in order:
    each is within the tolerance of the 64-bit form, and within twice that of the other."""
    q, kc, vc, bt, sl, scale = make([700, 33, 1999, 16], 32, 8, 128, 16, torch.bfloat16)
    out, plain = check(kernels, q, kc, vc, bt, sl, scale), torch.empty_like(q)
    kernels.paged_attention_forward(plain, q, kc, vc, bt, sl, scale, 16, bt.size(1))
    want, A, l = shaped_oracle.attend_single(q, kc, vc, bt, sl, scale)
    tol = shaped_oracle.attention_tolerance(want, A, l, 1999, q.dtype, float(vc.abs().max()))
    assert ((out.double() - plain.double()).abs() <= 2 * tol).all()


def test_scores_far_beyond_the_cap(kernels):
    """Scores of hundreds of caps, both signs: every probability of a row saturates, ties of +-cap share the weight."""
    q, kc, vc, bt, sl, scale = make([300, 64], 12, 2, 128, 16, torch.bfloat16, gain=100.0)
    check(kernels, q, kc, vc, bt, sl, scale, 8.0)


def test_infinite_keys_are_capped(kernels):
    """A key of +-inf along the query gives a score of +-cap, a finite row."""
    q, kc, vc, bt, sl, scale = make([100], 2, 2, 64, 16, torch.float16)
    q.fill_(1.0)
    kc[bt[0, 2].long(), :, 5, 3] = float("inf")
    kc[bt[0, 0].long(), :, :, 3] = float("-inf")
    check(kernels, q, kc, vc, bt, sl, scale, 4.0)


def test_uncapped_minus_infinity_scores_are_left_out(kernels):
    """The first tiles of a row score -inf (keys of -inf): they weigh nothing, as in the formula."""
    q, kc, vc, bt, sl, scale = make([100], 2, 2, 64, 16, torch.float16)
    q.fill_(1.0)
    for page in (0, 1, 2):
        kc[bt[0, page].long(), :, :, 3] = float("-inf")
    check(kernels, q, kc, vc, bt, sl, scale)
    check(kernels, q, kc, vc, bt, sl, scale, max_ctas=100)


def test_strided_tables_cache_views_and_rows_behind_the_batch(kernels):
    lens = [257, 31, 90]
    q, kc, vc, bt, sl, scale = make(lens, 12, 2, 128, 16, torch.float16)
    pool = torch.full((kc.size(0), 2, *kc.shape[1:]), float("nan"), dtype=kc.dtype, device=DEV)
    pool[:, 0], pool[:, 1] = kc, vc                              # K and V of a block side by side: a block stride of two blocks
    wide = torch.full((3, bt.size(1) + 5), 10 ** 6, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + bt.size(1)] = bt
    view = wide[:, 2:2 + bt.size(1)]
    guard = torch.full((5, 12, 128), 7.0, dtype=q.dtype, device=DEV)
    out = guard[:3]
    kernels.paged_scored_attention(out, q, pool[:, 0], pool[:, 1], view, sl, scale, 16, bt.size(1), score_cap=9.0, window=50)
    torch.cuda.synchronize()
    want, A, l = shaped_oracle.attend_single(q, kc, vc, bt, sl, scale, 9.0, None, 50)
    assert ((out.double() - want).abs() <= shaped_oracle.attention_tolerance(want, A, l, 257, q.dtype, float(vc.abs().max()))).all()
    assert (guard[3:] == 7.0).all()


def test_pool_beyond_32_bit_offsets(kernels):
    """Pages whose element offset passes 2^31."""
    lens, block = [200, 37], 16
    q, kc, vc, bt, sl, scale = make(lens, 32, 8, 128, block, torch.bfloat16)
    blocks = (1 << 31) // (8 * block * 128) + 64
    big_k, big_v = (torch.empty(blocks, 8, block, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    at = blocks - 1 - torch.arange(kc.size(0), device=DEV)
    big_k[at], big_v[at] = kc, vc
    far = at[bt.long()].to(torch.int32)
    out, near = torch.empty_like(q), torch.empty_like(q)
    kernels.paged_scored_attention(out, q, big_k, big_v, far, sl, scale, block, far.size(1), score_cap=30.0, window=64)
    kernels.paged_scored_attention(near, q, kc, vc, bt, sl, scale, block, bt.size(1), score_cap=30.0, window=64)
    assert torch.equal(out, near)


def test_bad_block_ids_are_flagged_and_skipped(kernels):
    q, kc, vc, bt, sl, scale = make([64, 64], 12, 2, 128, 16, torch.float16)
    bt[1, 3] = 10 ** 6
    out = torch.empty_like(q)
    kernels.paged_scored_attention(out, q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=30.0)
    assert kernels.check_status(raise_on_error=False) & 1
    bt[1, 3] = 0
    sl[1] = 10 ** 6                                              # beyond the table: clamped and flagged
    kernels.paged_scored_attention(out, q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=30.0)
    assert kernels.check_status(raise_on_error=False) == 2
    assert kernels.check_status() == 0


def test_another_stream_and_repeated_calls(kernels):
    lens = [3000, 17, 800, 1201]
    q, kc, vc, bt, sl, scale = make(lens, 32, 8, 128, 16, torch.bfloat16)
    first = check(kernels, q, kc, vc, bt, sl, scale, 50.0, None, 2000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.empty_like(q) for _ in range(6)]
    with torch.cuda.stream(side):
        for o in outs[::2]:
            kernels.paged_scored_attention(o, q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=50.0, window=2000)
    for o in outs[1::2]:
        kernels.paged_scored_attention(o, q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=50.0, window=2000)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, first)


def test_two_graphs_of_one_stream_replayed_side_by_side(kernels):
    """Each capture has scratch of its own: two graphs captured on the same stream may overlap."""
    lens = [[5000, 2000, 900, 31], [777, 4444, 3]]
    state = [make(n, 32, 8, 128, 16, torch.bfloat16, seed=i) for i, n in enumerate(lens)]
    want = [check(kernels, *st, 50.0) for st in state]
    graphs, outs = [], [torch.empty_like(w) for w in want]
    cap_stream = torch.cuda.Stream()
    for st, o in zip(state, outs):
        q, kc, vc, bt, sl, scale = st
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap_stream):
            kernels.paged_scored_attention(o, q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=50.0)
            kernels.paged_scored_attention(o, q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=50.0)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    # lengths change in place between replays
    state[0][4].copy_(torch.tensor([64, 1, 0, 31], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    q, kc, vc, bt, sl, scale = state[0]
    ref, A, l = shaped_oracle.attend_single(q, kc, vc, bt, sl, scale, 50.0)
    assert ((outs[0].double() - ref).abs() <= shaped_oracle.attention_tolerance(ref, A, l, 64, q.dtype, float(vc.abs().max()))).all()


@pytest.mark.parametrize("change,match", [
    (dict(score_cap=-1.0), "score_cap"), (dict(score_cap=float("nan")), "score_cap"), (dict(score_cap=float("inf")), "score_cap"),
    (dict(score_cap=1e-38), "cap"), (dict(window=-1), "window"), (dict(window=2.5), "window"),
    (dict(distance_slopes="short"), "distance_slopes"), (dict(distance_slopes="half"), "distance_slopes"),
    (dict(distance_slopes="cpu"), "distance_slopes"), (dict(max_ctas=-1), "max_ctas"),
])
def test_refusals(kernels, change, match):
    q, kc, vc, bt, sl, scale = make([20, 3], 12, 2, 128, 16, torch.float16)
    named = {"short": torch.ones(11, device=DEV), "half": torch.ones(12, device=DEV, dtype=torch.float16), "cpu": torch.ones(12)}
    change = {k: named[v] if isinstance(v, str) else v for k, v in change.items()}
    with pytest.raises(RuntimeError, match=match):
        kernels.paged_scored_attention(torch.empty_like(q), q, kc, vc, bt, sl, scale, 16, bt.size(1), **change)


def test_refusals_of_tensors(kernels):
    q, kc, vc, bt, sl, scale = make([20, 3], 12, 2, 128, 16, torch.float16)
    call = lambda out=None, q_=q, k=kc, v=vc, t=bt, n=sl, b=16, w=bt.size(1): kernels.paged_scored_attention(  # noqa: E731
        torch.empty_like(q_) if out is None else out, q_, k, v, t, n, scale, b, w)
    for bad in (dict(t=bt.long()), dict(n=sl.long()), dict(k=kc.bfloat16()), dict(k=kc[:, :1]), dict(q_=q[:, :11].contiguous()), dict(b=8),
                dict(w=bt.size(1) + 1), dict(w=0), dict(n=sl[:1]), dict(t=bt[:1]), dict(q_=q.transpose(0, 1)), dict(out=torch.empty_like(q).float()),
                dict(q_=q.cpu()), dict(t=bt.t().contiguous().t()), dict(q_=q[..., :64].contiguous())):
        if bad.get("t") is not None and bad["t"].stride(-1) == 1 and bad["t"].dtype == torch.int32 and bad["t"].size(0) == 2:
            continue                                            # a table of one column: its transpose is itself
        with pytest.raises(RuntimeError):
            call(**bad)
    with pytest.raises(RuntimeError, match="takes tensors"):
        kernels.paged_scored_attention(None, q, kc, vc, bt, sl, scale, 16, bt.size(1))


@pytest.mark.parametrize("scale", [-0.1, float("nan"), float("inf")])
def test_scales_that_are_refused(kernels, scale):
    q, kc, vc, bt, sl, _ = make([20, 3], 12, 2, 128, 16, torch.float16)
    with pytest.raises(RuntimeError, match="scale"):
        kernels.paged_scored_attention(torch.empty_like(q), q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=5.0)


def test_a_scale_of_zero_weighs_every_key_alike(kernels):
    q, kc, vc, bt, sl, _ = make([20, 300], 12, 2, 128, 16, torch.float16)
    check(kernels, q, kc, vc, bt, sl, 0.0, 5.0, None, 100)


def test_more_sequences_than_a_launch_takes(kernels):
    lens = [1 + i % 70 for i in range(5000)]
    q, kc, vc, bt, sl, scale = make(lens, 4, 2, 64, 16, torch.float16)
    check(kernels, q, kc, vc, bt, sl, scale, 6.0, slopes_for(4), 33)


def test_a_larger_call_after_a_smaller_one_in_one_capture(kernels):
    """The capture's scratch grows with its calls: more sequences need more cleared tickets."""
    small = make([3000, 2500], 32, 8, 128, 16, torch.bfloat16)
    large = make([700 + 13 * i for i in range(64)], 32, 8, 128, 16, torch.bfloat16, seed=1)
    want = [check(kernels, *st, 50.0, max_ctas=140) for st in (small, large)]
    outs = [torch.empty_like(w) for w in want]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for st, o in zip((small, large, small), outs + [outs[0]]):
            q, kc, vc, bt, sl, scale = st
            kernels.paged_scored_attention(o, q, kc, vc, bt, sl, scale, 16, bt.size(1), score_cap=50.0, max_ctas=140)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_workspaces_are_dropped_and_made_again(kernels):
    q, kc, vc, bt, sl, scale = make([3000, 17], 32, 8, 128, 16, torch.bfloat16)
    want = check(kernels, q, kc, vc, bt, sl, scale, 50.0, max_ctas=140)
    from nanopd_b200 import paged_kernels
    paged_kernels.release_workspaces(DEV)
    assert torch.equal(check(kernels, q, kc, vc, bt, sl, scale, 50.0, max_ctas=140), want)


@pytest.mark.parametrize("window", [0, 100000])
def test_very_long_contexts(kernels, window):
    lens = [150001, 7, 99999]
    q, kc, vc, bt, sl, scale = make(lens, 4, 1, 128, 16, torch.bfloat16, gain=2.0)
    check(kernels, q, kc, vc, bt, sl, scale, 30.0, None, window)
    check(kernels, q, kc, vc, bt, sl, scale, 0.0, slopes_for(4) * 0.01, window)
