"""CPU: threads that share a stream.  The operators over shared scratch hold the stream from the choice of the scratch to their
last launch; the launches are stand-ins that take their time."""
import threading
import time
from types import SimpleNamespace

import pytest
import torch

from nanopd_b200 import paged_kernels

HQ, D, BS = 4, 64, 16


def call(op, rows):
    q = torch.zeros(rows, HQ, D, dtype=torch.float16)
    kc = torch.zeros(4, 2, BS, D, dtype=torch.float16)
    bt, sl = torch.zeros(rows, 2, dtype=torch.int32), torch.ones(rows, dtype=torch.int32)
    if op == "scored":
        paged_kernels.paged_scored_attention(q, q, kc, kc, bt, sl, 0.1, BS, 2, score_cap=5.0)
    else:
        paged_kernels.paged_shared_prefix_attention(q, q, kc, kc, bt, sl, torch.tensor([0, rows], dtype=torch.int32), sl[:1], 0.1, BS, 2)


@pytest.fixture()
def steps(monkeypatch):
    """The steps of every call: ("scratch", thread) when it has chosen its buffer, ("in" / "out", thread) around its launches."""
    done = []
    me = lambda: threading.current_thread().name  # noqa: E731
    dev = torch.device("cpu")
    check = lambda name, out, q, *a: (dev, q.size(0), HQ, 2, D, BS, 4, 2 * BS * D, 2, 2)  # noqa: E731
    monkeypatch.setattr(paged_kernels, "_check_single_token_call", check)
    monkeypatch.setattr(paged_kernels, "_C", SimpleNamespace(npd_decode_workspace_bytes=lambda *a: 1024 * a[0],
                                                             npd_shared_prefix_workspace_bytes=lambda *a: 1024 * a[0]))
    monkeypatch.setattr(paged_kernels, "_raw_stream", lambda index: STREAM.get(me(), 7))
    monkeypatch.setattr(paged_kernels, "_status_addresses", {None: 64})
    for name in ("_scored_plans", "_shared_plans", "_scratch_locks"):
        monkeypatch.setattr(paged_kernels, name, {})

    def scratch(index, handle, need, cleared):
        done.append(("scratch", me()))
        time.sleep(0.002)
        return 256, need

    def launch(op, pack, *args):
        done.append(("in", me()))
        time.sleep(0.005)
        done.append(("out", me()))

    monkeypatch.setattr(paged_kernels, "_scratch_for", scratch)
    monkeypatch.setattr(paged_kernels, "_packed_op", launch)
    return done


STREAM = {}


@pytest.mark.parametrize("ops", [("shared", "shared"), ("shared", "scored"), ("scored", "scored")])
def test_calls_on_one_stream_do_not_interleave(steps, ops):
    STREAM.clear()
    threads = [threading.Thread(target=lambda o=o, i=i: [call(o, 2 + i) for _ in range(5)], name=f"t{i}") for i, o in enumerate(ops)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(steps) == 30
    for i in range(0, 30, 3):
        assert [s for s, _ in steps[i:i + 3]] == ["scratch", "in", "out"] and len({t for _, t in steps[i:i + 3]}) == 1


def test_streams_do_not_wait_for_one_another(steps, monkeypatch):
    STREAM.clear()
    STREAM.update(a=1, b=2)
    both = threading.Barrier(2)
    met = []
    monkeypatch.setattr(paged_kernels, "_packed_op", lambda *args: met.append(both.wait(timeout=20)))
    threads = [threading.Thread(target=call, args=("shared", 3), name=n) for n in ("a", "b")]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(met) == [0, 1]


def test_workspaces_are_released_between_calls_only(steps, monkeypatch):
    STREAM.clear()
    inside, checked = threading.Event(), []
    monkeypatch.setattr(paged_kernels, "_scratch", {(None, 7): torch.zeros(1)})
    monkeypatch.setattr(paged_kernels, "_scratch_at", {(None, 7): (256, 1)})
    monkeypatch.setattr(paged_kernels, "_captured_scratch", {})
    monkeypatch.setattr(paged_kernels, "_workspaces", {})
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)

    def launch(*args):
        inside.set()
        time.sleep(0.05)
        checked.append((None, 7) in paged_kernels._scratch)

    monkeypatch.setattr(paged_kernels, "_packed_op", launch)
    t = threading.Thread(target=call, args=("shared", 3))
    t.start()
    inside.wait(20)
    paged_kernels.release_workspaces()
    t.join()
    assert checked == [True] and not paged_kernels._scratch and not paged_kernels._scratch_at
