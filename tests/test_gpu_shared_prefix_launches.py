"""GPU: the plan, prefix and tail launches of the shared-prefix operator, on batches that the operator would answer in one
launch if the number of CTAs were not limited."""
import os
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import test_gpu_shared_prefix as one_launch
from nanopd_b200 import paged_kernels
from test_gpu_shared_prefix import call, check, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture()
def limited(kernels):
    """The operators with the number of CTAs limited, which switches the one-launch form off."""
    class Limited:
        @staticmethod
        def paged_shared_prefix_attention(*args, **kw):
            kernels.paged_shared_prefix_attention(*args, **{"max_ctas": 140, **kw})

        def __getattr__(self, name):
            return getattr(kernels, name)

    return Limited()


@pytest.mark.parametrize("shared", [0, 15, 16, 17, 31, 32, 63, 64, 65, 127, 128, 129, 255, 1000, 4112])
def test_lengths_of_the_prefix(limited, shared):
    one_launch.test_lengths_of_the_prefix(limited, shared)


@pytest.mark.parametrize("case", ["test_prefix_that_is_the_whole_of_some_sequences", "test_idle_slots_in_a_group", "test_large_scores",
                                  "test_groups_that_do_not_ascend_share_nothing", "test_agrees_with_the_plain_operator_and_repeats_bit_for_bit",
                                  "test_rows_behind_the_batch_and_strided_tables", "test_graphs_with_changing_lengths_and_side_streams",
                                  "test_many_sequences_and_many_groups"])
def test_cases_of_the_one_launch_form(limited, case):
    """Prefixes that the shortest sequence cuts, offsets that do not ascend, replays of one graph with other lengths, graphs
    replayed side by side: through plan, prefix pass and tail."""
    getattr(one_launch, case)(limited)


@pytest.mark.parametrize("hq,hkv,d", [(32, 1, 128), (16, 16, 64), (16, 2, 256)])
@pytest.mark.parametrize("max_ctas", [1, 2, 9])
def test_hundreds_of_short_pieces_to_a_cta(kernels, hq, hkv, d, max_ctas):
    """Prefixes of one key tile and groups of two: items that give the second query tile no work follow one another."""
    state = make([(16 * (1 + i % 4), [1 + (i + j) % 9 for j in range(2)]) for i in range(150)], hq, hkv, d, 16, torch.bfloat16)
    first = check(kernels, state, max_ctas=max_ctas)
    for _ in range(5):
        assert torch.equal(check(kernels, state, max_ctas=max_ctas), first)


@pytest.mark.parametrize("idle", [(0,), (0, 1), (2,), (0, 3), (1, 2, 3)])
@pytest.mark.parametrize("max_ctas", [0, 140])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (12, 2, 64), (16, 2, 256)])
def test_idle_slots_whose_rows_name_other_pages(kernels, hq, hkv, d, max_ctas, idle):
    """An empty slot's table row is parked on a page of NaN (and, behind it, names no page at all): neither the group's other
    sequences nor the status word see it."""
    q, kc, vc, bt, sl, go, sh = make([(96, [5, 8]), (512, [9, 30, 100, 7]), (64, [3, 4])], hq, hkv, d, 16, torch.bfloat16)
    used = set(bt[:, :].flatten().tolist())
    parked = next(i for i in range(kc.size(0)) if i not in used or bool(torch.isnan(kc[i]).all()))
    kc[parked], vc[parked] = float("nan"), float("nan")
    for i in idle:
        sl[2 + i] = 0
        bt[2 + i] = -5
        bt[2 + i, 0] = parked
    out = check(kernels, (q, kc, vc, bt, sl, go, sh), max_ctas=max_ctas)
    for i in idle:
        assert (out[2 + i] == 0).all()


@pytest.mark.parametrize("max_ctas", [0, 140, 2])
def test_keys_whose_scores_are_minus_infinity(kernels, max_ctas):
    """Pages of the prefix, whole pieces of it and all own tokens of a sequence may score -inf: they weigh nothing, and the rest
    of the row is what it is without them."""
    q, kc, vc, bt, sl, go, sh = make([(640, [5, 20, 100, 33]), (256, [3, 40])], 12, 2, 128, 16, torch.float16)
    q.fill_(1.0)
    kc[bt[0, :9].long(), :, :, 3] = float("-inf")               # more than the first key tile of the first group
    kc[bt[0, 20:37].long(), :, :, 3] = float("-inf")
    kc[bt[4, 8:16].long(), :, :, 7] = float("-inf")             # the whole second tile of the second
    kc[bt[1, 40:42].long(), :, :, 9] = float("-inf")            # every own token of sequence 1
    check(kernels, (q, kc, vc, bt, sl, go, sh), max_ctas=max_ctas)
    kc[bt[4, :16].long(), :, :, 7] = float("-inf")              # the whole prefix of the second group
    check(kernels, (q, kc, vc, bt, sl, go, sh), max_ctas=max_ctas)


def test_threads_on_one_stream(kernels):
    """Four threads on the default stream, each with its own batch (of its own size, so that the scratch grows between the
    calls): three launches a call, none of them another call's."""
    paged_kernels.release_workspaces()
    states = [make([(64 * (i + 1), [5 + i, 40, 7]), (512, [3 + j for j in range(4 + 20 * i)])], 12, 2, 128, 16, torch.float16, seed=i) for i in range(4)]
    outs, errors = [[] for _ in states], []

    def work(i):
        try:
            for _ in range(40):
                out = torch.full_like(states[i][0], float("nan"))
                call(kernels, out, *states[i], max_ctas=140)
                outs[i].append(out)
        except Exception as e:                                  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(states))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for s, got in zip(states, outs):
        want = check(kernels, s, max_ctas=140)
        assert all(torch.equal(o, want) for o in got)


def test_an_odd_number_of_stages_of_a_cta(kernels):
    """Five warps of one stage each leave the barriers' end in the middle of a 16-byte piece."""
    here = Path(__file__).resolve()
    env = dict(os.environ, NPD_DECODE_WARPS="5", NPD_DECODE_STAGES="1")
    res = subprocess.run([sys.executable, "-m", "pytest", str(here.with_name("test_gpu_shared_prefix.py")), "-q", "-x", "-p", "no:cacheprovider",
                          "-k", "test_shapes"], env=env, capture_output=True, text=True, timeout=600, cwd=str(here.parents[1]))
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-2000:]
