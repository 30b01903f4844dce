"""GPU: prompt attention with shaped scores (cap, distance bias, window) against a plain form in 64 bits."""
import pytest
import torch

from oracle import shaped_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(chunks, hq, hkv, d, block, dtype, seed=0, gain=1.0, spare=2):
    """``chunks``: (start, tokens).  Pages in random order, one table row per chunk; queries packed."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    need = [-(-(s + n) // block) for s, n in chunks]
    perm = torch.randperm(sum(need) + spare, generator=gen, device=DEV).to(torch.int32)
    bt = torch.zeros(len(chunks), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)  # noqa: E731
    total = sum(n for _, n in chunks)
    return r(total, hq, d) * gain, r(sum(need) + spare, hkv, block, d), r(sum(need) + spare, hkv, block, d), bt


def poison(kc, vc, bt, chunks, window, value=float("nan")):
    block = kc.size(2)
    seen = torch.zeros(kc.size(0), block, dtype=torch.bool)
    bt_cpu = bt.cpu()
    for c, (start, n) in enumerate(chunks):
        lo = max(0, start - window + 1) if window else 0
        for j in range(lo, start + n):
            seen[int(bt_cpu[c, j // block]), j % block] = True
        if n:
            bt_cpu[c, :lo // block] = -9
    hide = (~seen).to(kc.device)
    kc.permute(0, 2, 1, 3)[hide] = value
    vc.permute(0, 2, 1, 3)[hide] = value
    bt.copy_(bt_cpu)


def slopes_for(hq):
    return torch.exp2(-8.0 * torch.arange(1, hq + 1, dtype=torch.float32, device=DEV) / hq)


def call(kernels, out, q, kc, vc, bt, chunks, scale, **kw):
    offs, at = [], 0
    for _, n in chunks:
        offs.append(at)
        at += n
    kernels.paged_scored_prefill_attention(out, q, kc, vc, bt, offs, [n for _, n in chunks], [s for s, _ in chunks], scale, kc.size(2),
                                           bt.size(1), **kw)


def check(kernels, q, kc, vc, bt, chunks, cap=0.0, slopes=None, window=0, **kw):
    scale = float(q.size(2)) ** -0.5
    out = torch.full_like(q, float("nan"))
    call(kernels, out, q, kc, vc, bt, chunks, scale, score_cap=cap, distance_slopes=slopes, window=window, **kw)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()
    v_max, at = float(vc[torch.isfinite(vc)].abs().max()), 0
    for c, (start, n) in enumerate(chunks):
        if n == 0:
            continue
        want, A, l = shaped_oracle.attend(q[at:at + n], kc, vc, bt[c], start, scale, cap, slopes, window)
        # a stale maximum lets a probability reach 2^8 before the row sum divides it away: subnormal steps stay those of 1
        tol = shaped_oracle.attention_tolerance(want, A, l, start + n, q.dtype, v_max)
        off = (out[at:at + n].double() - want).abs()
        assert (off <= tol).all(), f"chunk {c}: worst {float((off / tol).max()):.2f} of the tolerance"
        at += n
    return out


SHAPES = [
    (12, 2, 128, 16, [(0, 1), (205, 23), (1, 77), (40, 130)]),
    (32, 8, 128, 16, [(0, 300), (512, 512), (63, 65), (64, 64)]),
    (16, 16, 64, 8, [(0, 257), (100, 129), (7, 1)]),
    (14, 2, 64, 32, [(31, 33), (0, 200)]),
    (8, 2, 256, 32, [(0, 130), (95, 70), (200, 1)]),
    (24, 8, 128, 4, [(3, 5), (60, 90)]),
    (40, 1, 128, 16, [(10, 40)]),
]
SCORES = [(50.0, False, 0), (0.0, True, 0), (0.0, False, 40), (30.0, True, 33), (20.0, False, 1), (0.0, True, 64), (5.0, True, 100000)]


@pytest.mark.parametrize("cap,bias,window", SCORES)
@pytest.mark.parametrize("hq,hkv,d,block,chunks", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_shapes_and_scores(kernels, dtype, hq, hkv, d, block, chunks, cap, bias, window):
    q, kc, vc, bt = make(chunks, hq, hkv, d, block, dtype, gain=3.0 if cap else 1.0)
    poison(kc, vc, bt, chunks, window)
    check(kernels, q, kc, vc, bt, chunks, cap, slopes_for(hq) if bias else None, window)


@pytest.mark.parametrize("window", [1, 17, 63, 64, 65, 127, 128, 129, 500, 1024, 5000])
def test_windows_over_a_long_prompt(kernels, window):
    chunks = [(0, 1500), (1300, 700), (4000, 100), (3999, 1), (0, 0)]
    q, kc, vc, bt = make(chunks, 16, 4, 128, 16, torch.bfloat16, gain=2.0)
    poison(kc, vc, bt, chunks, window)
    check(kernels, q, kc, vc, bt, chunks, 50.0, None, window)
    check(kernels, q, kc, vc, bt, chunks, 0.0, slopes_for(16), window, max_ctas=7)


def test_more_chunks_than_a_launch_takes(kernels):
    chunks = [(7 * i, 3 + i % 9) for i in range(70)]
    q, kc, vc, bt = make(chunks, 8, 2, 128, 16, torch.float16)
    check(kernels, q, kc, vc, bt, chunks, 10.0, slopes_for(8), 100)


def test_without_shaping_agrees_with_the_plain_operator(kernels):
    chunks = [(0, 700), (128, 300)]
    q, kc, vc, bt = make(chunks, 32, 8, 128, 16, torch.bfloat16)
    out = check(kernels, q, kc, vc, bt, chunks)
    plain = torch.empty_like(q)
    kernels.paged_prefill_attention(plain, q, kc, vc, bt, [0, 700], [700, 300], [0, 128], 128 ** -0.5, 16, bt.size(1))
    assert (out.float() - plain.float()).abs().max() <= 2 ** -7


@pytest.mark.parametrize("gain", [0.001, 20.0, 100.0])
def test_both_branches_of_the_cap(kernels, gain):
    """Scores far below the cap, around it, and hundreds of caps away, in the same launch."""
    chunks = [(0, 200), (90, 64)]
    q, kc, vc, bt = make(chunks, 12, 2, 128, 16, torch.bfloat16)
    q[::3] *= gain
    check(kernels, q, kc, vc, bt, chunks, 8.0)


def test_infinite_scores(kernels):
    chunks = [(0, 150)]
    q, kc, vc, bt = make(chunks, 2, 2, 64, 16, torch.float16)
    q.fill_(1.0)
    kc[bt[0, 2].long(), :, 5, 3] = float("inf")
    kc[bt[0, 4].long(), :, 1, 3] = float("-inf")
    check(kernels, q, kc, vc, bt, chunks, 4.0)
    # uncapped: whole half-steps of -inf weigh nothing for the rows behind them
    kc[bt[0, 2].long(), :, 5, 3] = 0.5
    for page in range(4):
        kc[bt[0, page].long(), :, :, 3] = float("-inf")
    scale, out = 0.125, torch.empty_like(q)
    call(kernels, out, q, kc, vc, bt, chunks, scale)
    want, A, l = shaped_oracle.attend(q[65:], kc, vc, bt[0], 65, scale)
    assert ((out[65:].double() - want).abs() <= shaped_oracle.attention_tolerance(want, A, l, 150, q.dtype, float(vc.abs().max()))).all()


def test_rows_outside_every_chunk_and_strided_tables(kernels):
    q, kc, vc, bt = make([(20, 30)], 12, 2, 128, 16, torch.float16)
    big_q = torch.randn(64, 12, 128, device=DEV).to(torch.float16)
    big_q[17:47] = q
    out = torch.full_like(big_q, 7.0)
    wide = torch.full((1, bt.size(1) + 3), -1, dtype=torch.int32, device=DEV)
    wide[:, :bt.size(1)] = bt
    kernels.paged_scored_prefill_attention(out, big_q, kc, vc, wide, [17], [30], [20], 128 ** -0.5, 16, bt.size(1), score_cap=9.0, window=25)
    want, A, l = shaped_oracle.attend(q, kc, vc, bt[0], 20, 128 ** -0.5, 9.0, None, 25)
    assert ((out[17:47].double() - want).abs() <= shaped_oracle.attention_tolerance(want, A, l, 50, q.dtype, float(vc.abs().max()))).all()
    assert (out[:17] == 7).all() and (out[47:] == 7).all()


def test_bad_block_ids_are_flagged(kernels):
    q, kc, vc, bt = make([(0, 60)], 12, 2, 128, 16, torch.float16)
    bt[0, 1] = 10 ** 6
    call(kernels, torch.empty_like(q), q, kc, vc, bt, [(0, 60)], 0.1, score_cap=5.0)
    assert kernels.check_status(raise_on_error=False) == 1


def test_streams_and_graphs(kernels):
    chunks = [(0, 900), (300, 500)]
    q, kc, vc, bt = make(chunks, 32, 8, 128, 16, torch.bfloat16)
    want = check(kernels, q, kc, vc, bt, chunks, 30.0, None, 400)
    graphs, outs, cap = [], [torch.empty_like(q) for _ in range(4)], torch.cuda.Stream()
    for o in outs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap):
            call(kernels, o, q, kc, vc, bt, chunks, 128 ** -0.5, score_cap=30.0, window=400)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in outs]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        for o, s in zip(outs[2:], streams[2:]):
            with torch.cuda.stream(s):
                call(kernels, o, q, kc, vc, bt, chunks, 128 ** -0.5, score_cap=30.0, window=400)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_refusals(kernels):
    q, kc, vc, bt = make([(0, 20), (4, 10)], 12, 2, 128, 16, torch.float16)

    def run(out=None, q_=q, k=kc, v=vc, t=bt, offs=(0, 20), toks=(20, 10), starts=(0, 4), b=16, w=bt.size(1), **kw):
        kernels.paged_scored_prefill_attention(torch.empty_like(q_) if out is None else out, q_, k, v, t, offs, toks, starts, 0.1, b, w, **kw)

    run()
    for kw in (dict(score_cap=-1.0), dict(score_cap=float("nan")), dict(window=-1), dict(window=1.5), dict(distance_slopes=torch.ones(11, device=DEV)),
               dict(distance_slopes=torch.ones(12)), dict(t=bt.long()), dict(t=bt[:1]), dict(offs=(0, 21)), dict(toks=(20, -1)), dict(starts=(0, -4)),
               dict(starts=(0, 10 ** 6)), dict(b=8), dict(w=bt.size(1) + 1), dict(k=kc.bfloat16()), dict(q_=q[:, :11].contiguous()), dict(q_=q.cpu()),
               dict(out=q.float()), dict(max_ctas=-1), dict(t=None), dict(toks=5), dict(k=kc[:, :, :8])):
        with pytest.raises(RuntimeError):
            run(**kw)


@pytest.mark.parametrize("scale", [-0.1, float("nan"), float("inf")])
def test_scales_that_are_refused(kernels, scale):
    q, kc, vc, bt = make([(0, 20)], 12, 2, 128, 16, torch.float16)
    with pytest.raises(RuntimeError, match="scale"):
        call(kernels, torch.empty_like(q), q, kc, vc, bt, [(0, 20)], scale, score_cap=5.0)


@pytest.mark.parametrize("cap", [1e-9, 1e-3, 1e9])
def test_caps_far_from_the_usual(kernels, cap):
    chunks = [(0, 200), (70, 40)]
    q, kc, vc, bt = make(chunks, 12, 2, 128, 16, torch.float16)
    if cap > 1:             # scores of 1e9 caps would need their 32 bits for themselves: the cap leaves these as they are
        out, plain = torch.empty_like(q), torch.empty_like(q)
        call(kernels, plain, q, kc, vc, bt, chunks, 128 ** -0.5)
        call(kernels, out, q, kc, vc, bt, chunks, 128 ** -0.5, score_cap=200.0)
        assert (out.float() - plain.float()).abs().max() <= 2 ** -8
    else:
        check(kernels, q, kc, vc, bt, chunks, cap)


@pytest.mark.parametrize("hq,hkv,d", [(24, 8, 128), (14, 2, 64), (12, 2, 128), (40, 1, 128)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_results_do_not_depend_on_what_ran_before(kernels, hq, hkv, d, cap):
    """Groups that do not divide 128 leave rows of a query tile unused: their leftovers (infinite, tiny, NaN) change nothing."""
    chunks = [(0, 300), (77, 130)]
    q, kc, vc, bt = make(chunks, hq, hkv, d, 16, torch.bfloat16, gain=2.0)
    full = make([(0, 2600)], 32, 8, d, 16, torch.bfloat16, seed=1)
    want = check(kernels, q, kc, vc, bt, chunks, cap)
    out, junk = torch.empty_like(q), torch.empty_like(full[0])
    for leftover in (float("inf"), 1e30, 0.0, float("nan")):
        full[0].fill_(leftover)                                  # every row of every query tile of this launch
        call(kernels, junk, *full, [(0, 2600)], d ** -0.5, score_cap=cap)
        call(kernels, out, q, kc, vc, bt, chunks, d ** -0.5, score_cap=cap)
        assert torch.equal(out, want)


@pytest.mark.parametrize("hq,hkv,d,block", [(64, 8, 128, 8), (32, 1, 128, 16), (8, 8, 64, 16), (16, 2, 256, 16)])
def test_many_items_of_a_single_key_tile(kernels, hq, hkv, d, block):
    """A short window makes every work item one key tile long: the producer runs as far ahead of the epilogue as it can."""
    chunks = [(0, 2775)]
    q, kc, vc, bt = make(chunks, hq, hkv, d, block, torch.bfloat16, gain=0.3)
    poison(kc, vc, bt, chunks, 6)
    want = check(kernels, q, kc, vc, bt, chunks, 50.0, slopes_for(hq), 6)
    out = torch.empty_like(q)
    for i in range(40):
        call(kernels, out, q, kc, vc, bt, chunks, d ** -0.5, score_cap=50.0, distance_slopes=slopes_for(hq), window=6, max_ctas=(0, 1, 5, 100)[i % 4])
        assert torch.equal(out, want)
