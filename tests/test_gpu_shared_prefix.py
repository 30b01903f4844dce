"""GPU: decode attention for batches that share prefixes against a plain form in 64 bits."""
import pytest
import torch

from oracle import shaped_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(groups, hq, hkv, d, block, dtype, seed=0, lead=(), trail=()):
    """``groups``: (shared tokens, own tokens of each sequence); ``lead``, ``trail``: lengths of sequences outside every group.
    A shared part that ends inside a page is followed by own tokens in that very page only for groups of whole pages, so the
    pages of a group's shared tokens are shared up to the last whole one and copied behind it."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rows, lens, offs, shared, total = [], [], [len(lead)], [], 0

    def fresh(n):
        nonlocal total
        total += n
        return list(range(total - n, total))

    for n in lead:
        rows.append(fresh(-(-n // block)))
        lens.append(n)
    for p, own in groups:
        head = fresh(p // block)
        for n in own:
            rows.append(head + fresh(-(-(p + n) // block) - len(head)))
            lens.append(p + n)
        offs.append(offs[-1] + len(own))
        shared.append(p // block * block)
    for n in trail:
        rows.append(fresh(-(-n // block)))
        lens.append(n)
    perm = torch.randperm(total + 1, generator=gen, device=DEV).to(torch.int32)
    bt = torch.zeros(len(rows), max(1, max(len(r) for r in rows)), dtype=torch.int32, device=DEV)
    for i, r in enumerate(rows):
        bt[i, :len(r)] = perm[torch.tensor(r, dtype=torch.long, device=DEV)] if r else 0
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)  # noqa: E731
    kc, vc = r(total + 1, hkv, block, d), r(total + 1, hkv, block, d)
    seen = torch.zeros(total + 1, block, dtype=torch.bool)
    bt_cpu = bt.cpu()
    for s, n in enumerate(lens):
        for j in range(n):
            seen[int(bt_cpu[s, j // block]), j % block] = True
    hide = (~seen).to(DEV)
    kc.permute(0, 2, 1, 3)[hide] = float("nan")
    vc.permute(0, 2, 1, 3)[hide] = float("nan")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return r(len(rows), hq, d), kc, vc, bt, i32(lens), i32(offs), i32(shared)


def call(kernels, out, q, kc, vc, bt, sl, go, sh, **kw):
    kernels.paged_shared_prefix_attention(out, q, kc, vc, bt, sl, go, sh, float(q.size(2)) ** -0.5, kc.size(2), bt.size(1), **kw)


def check(kernels, state, **kw):
    q, kc, vc, bt, sl, go, sh = state
    out = torch.full_like(q, float("nan"))
    call(kernels, out, *state, **kw)
    torch.cuda.synchronize()
    want, A, l = shaped_oracle.attend_single(q, kc, vc, bt, sl, float(q.size(2)) ** -0.5)
    tol = shaped_oracle.attention_tolerance(want, A, l, int(sl.max()), q.dtype, float(vc[torch.isfinite(vc)].abs().max()))
    off = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (off <= tol).all(), f"worst {float((off / tol).max()):.2f} of the tolerance"
    return out


@pytest.mark.parametrize("hq,hkv,d,block", [(32, 8, 128, 16), (12, 2, 128, 16), (16, 16, 64, 8), (14, 2, 64, 32), (8, 2, 256, 32), (40, 2, 128, 16),
                                            (16, 1, 256, 16), (24, 8, 128, 4), (128, 1, 64, 16)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_shapes(kernels, dtype, hq, hkv, d, block):
    groups = [(640, [1, 17, 300, 16]), (96, [5, 5]), (2000, [33] * 9), (64, [700]), (0, [40, 3])]
    state = make(groups, hq, hkv, d, block, dtype, lead=(70,), trail=(0, 129))
    check(kernels, state)
    check(kernels, state, max_ctas=13)


@pytest.mark.parametrize("shared", [0, 15, 16, 17, 31, 32, 63, 64, 65, 127, 128, 129, 255, 1000, 4112])
def test_lengths_of_the_prefix(kernels, shared):
    """``shared_lens`` may end inside a page or a tile: what no whole tile holds is read per sequence."""
    state = list(make([(shared, [1, 2, 16, 40, 100])], 12, 2, 128, 16, torch.float16))
    check(kernels, state)
    state[6] = torch.tensor([max(0, shared - 5)], dtype=torch.int32, device=DEV)      # fewer tokens than the tables share
    check(kernels, state)


def test_prefix_that_is_the_whole_of_some_sequences(kernels):
    """All of the shortest sequence's tokens are shared: the last tile stays with the sequences, every row is written."""
    for own in ([16, 0, 5], [0, 0, 0], [0, 64]):
        q, kc, vc, bt, sl, go, sh = make([(512, own)], 32, 8, 128, 16, torch.bfloat16)
        check(kernels, (q, kc, vc, bt, sl, go, sh))
        check(kernels, (q, kc, vc, bt, sl, go, torch.full_like(sh, 10 ** 6)))         # a claim beyond the shortest sequence is cut


def test_idle_slots_in_a_group(kernels):
    q, kc, vc, bt, sl, go, sh = make([(512, [9, 30, 100, 7])], 32, 8, 128, 16, torch.bfloat16)
    sl[0], sl[2] = 0, 0
    out = check(kernels, (q, kc, vc, bt, sl, go, sh))
    assert (out[0] == 0).all() and (out[2] == 0).all()
    sl.zero_()
    assert (check(kernels, (q, kc, vc, bt, sl, go, sh)) == 0).all()


def test_many_sequences_and_many_groups(kernels):
    check(kernels, make([(2048, [1 + i % 50 for i in range(200)])], 32, 8, 128, 16, torch.bfloat16))
    check(kernels, make([(48 + 16 * (i % 7), [1 + j for j in range(1 + i % 4)]) for i in range(150)], 8, 2, 128, 16, torch.float16))


def test_large_scores(kernels):
    """The prefix holds, or does not hold, nearly all of a row's weight."""
    q, kc, vc, bt, sl, go, sh = make([(300, [50, 7, 90])], 12, 2, 128, 16, torch.float16)
    check(kernels, (q * 12, kc, vc, bt, sl, go, sh))
    for scale in (1e-2, 5.0):
        k2 = kc.clone()
        k2[bt[0, :18].long()] *= scale
        check(kernels, (q * 4, k2, vc, bt, sl, go, sh))


def test_groups_that_do_not_ascend_share_nothing(kernels):
    q, kc, vc, bt, sl, go, sh = make([(256, [3, 4]), (128, [5, 6])], 12, 2, 128, 16, torch.float16)
    for bad in ([0, 3, 2], [-1, 2, 4], [0, 2, 99], [4, 2, 0]):
        check(kernels, (q, kc, vc, bt, sl, torch.tensor(bad, dtype=torch.int32, device=DEV), sh))
        assert kernels.check_status(raise_on_error=False) == 2
    check(kernels, (q, kc, vc, bt, sl, go, torch.tensor([-5, 128], dtype=torch.int32, device=DEV)))
    assert kernels.check_status(raise_on_error=False) == 2
    bt[0, 3] = 10 ** 6
    call(kernels, torch.empty_like(q), q, kc, vc, bt, sl, go, sh)
    assert kernels.check_status(raise_on_error=False) == 1


def test_agrees_with_the_plain_operator_and_repeats_bit_for_bit(kernels):
    state = make([(1500, [20, 300, 7, 64, 1000])], 32, 8, 128, 16, torch.bfloat16)
    first = check(kernels, state)
    q, kc, vc, bt, sl, go, sh = state
    plain = torch.empty_like(q)
    kernels.paged_attention_forward(plain, q, kc, vc, bt, sl, 128 ** -0.5, 16, bt.size(1))
    assert (plain.float() - first.float()).abs().max() <= 2 ** -7
    for _ in range(5):
        assert torch.equal(check(kernels, state), first)


def test_rows_behind_the_batch_and_strided_tables(kernels):
    q, kc, vc, bt, sl, go, sh = make([(256, [3, 40, 70])], 12, 2, 128, 16, torch.float16)
    wide = torch.full((3, bt.size(1) + 5), 10 ** 6, dtype=torch.int32, device=DEV)
    wide[:, 1:1 + bt.size(1)] = bt
    guard = torch.full((5, 12, 128), 7.0, dtype=q.dtype, device=DEV)
    call(kernels, guard[:3], q, kc, vc, wide[:, 1:1 + bt.size(1)], sl, go, sh)
    assert torch.equal(guard[:3], check(kernels, (q, kc, vc, bt, sl, go, sh))) and (guard[3:] == 7).all()


def test_graphs_with_changing_lengths_and_side_streams(kernels):
    states = [make([(1024, [20, 300, 7]), (64, [3, 5])], 32, 8, 128, 16, torch.bfloat16, seed=i) for i in range(2)]
    want = [check(kernels, s) for s in states]
    cap, graphs, outs = torch.cuda.Stream(), [], [torch.empty_like(w) for w in want]
    for s, o in zip(states, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap):
            call(kernels, o, *s)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    eager = torch.empty_like(want[0])
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            call(kernels, eager, *states[0])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])
    q, kc, vc, bt, sl, go, sh = states[0]
    sl.copy_(torch.tensor([1025, 1100, 0, 60, 67], dtype=torch.int32))
    sh.copy_(torch.tensor([512, 48], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], check(kernels, states[0]))


def test_refusals(kernels):
    q, kc, vc, bt, sl, go, sh = make([(256, [3, 40, 70])], 12, 2, 128, 16, torch.float16)

    def run(out=None, q_=q, k=kc, t=bt, n=sl, g=go, s=sh, b=16, w=bt.size(1), **kw):
        kernels.paged_shared_prefix_attention(torch.empty_like(q_) if out is None else out, q_, k, vc, t, n, g, s, 0.1, b, w, **kw)

    run()
    for kw in (dict(g=go.long()), dict(s=sh.long()), dict(g=go[:1]), dict(g=go.cpu()), dict(s=sh[:0]), dict(g=go[None]), dict(t=bt.long()), dict(n=sl[:2]),
               dict(b=8), dict(w=0), dict(k=kc.bfloat16()), dict(q_=q.cpu()), dict(out=q.float()), dict(max_ctas=70000), dict(g=None),
               dict(s=torch.zeros(4097, dtype=torch.int32, device=DEV), g=torch.zeros(4098, dtype=torch.int32, device=DEV)),
               dict(q_=q.float())):
        with pytest.raises(RuntimeError):
            run(**kw)
    kernels.paged_shared_prefix_attention(q[:0], q[:0], kc, vc, bt[:0], sl[:0], go, sh, 0.1, 16, bt.size(1))


@pytest.mark.parametrize("scale", [-0.1, float("nan"), float("inf")])
def test_scales_that_are_refused(kernels, scale):
    q, kc, vc, bt, sl, go, sh = make([(256, [3, 40, 70])], 12, 2, 128, 16, torch.float16)
    with pytest.raises(RuntimeError, match="scale"):
        kernels.paged_shared_prefix_attention(torch.empty_like(q), q, kc, vc, bt, sl, go, sh, scale, 16, bt.size(1))


def test_the_largest_batches(kernels):
    """4096 groups of one, two and three, and a batch that takes two sub-batches of the tail."""
    groups = [(16 * (i % 3), [1 + (i + j) % 20 for j in range(1 + i % 3)]) for i in range(4096)]
    state = make(groups, 4, 1, 64, 16, torch.float16)
    q, kc, vc, bt, sl, go, sh = state
    assert q.size(0) > 8000
    out = torch.full_like(q, float("nan"))
    call(kernels, out, *state)
    plain = torch.empty_like(q)
    kernels.paged_attention_forward(plain, q, kc, vc, bt, sl, 0.125, 16, bt.size(1))
    assert (out.float() - plain.float()).abs().max() <= 2 ** -9
    state = make([(1600, [1 + i % 30 for i in range(4100)])], 4, 1, 64, 16, torch.float16)
    q, kc, vc, bt, sl, go, sh = state
    out, plain = torch.full_like(q, float("nan")), torch.empty_like(q)
    call(kernels, out, *state)
    kernels.paged_attention_forward(plain, q, kc, vc, bt, sl, 0.125, 16, bt.size(1))
    assert (out.float() - plain.float()).abs().max() <= 2 ** -9


@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 256), (32, 8, 128), (16, 16, 64)])
def test_prefixes_that_end_inside_a_tile_many_pieces_to_a_cta(kernels, hq, hkv, d):
    """Eleven groups whose prefixes end inside a key tile; few CTAs, so that one works through many pieces."""
    groups = [(2000 + 16 * (3 * i % 8) + 64 * i, [1 + (7 * i + j) % 90 for j in range(9 + i)]) for i in range(11)]
    state = make(groups, hq, hkv, d, 16, torch.bfloat16)
    first = check(kernels, state)
    few = check(kernels, state, max_ctas=5)
    for _ in range(10):
        assert torch.equal(check(kernels, state), first)
        assert torch.equal(check(kernels, state, max_ctas=5), few)


@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (12, 1, 64), (4, 1, 256)])
def test_a_long_prefix_in_more_pieces_than_a_warp_has_lanes(kernels, hq, hkv, d):
    """One item whose key tiles go to every SM: a row is joined from more than a hundred pieces."""
    state = make([(30000, [5, 100, 1, 33, 64, 17, 2, 300])], hq, hkv, d, 16, torch.float16)
    first = check(kernels, state)
    assert torch.equal(check(kernels, state), first)
    check(kernels, state, max_ctas=40)
