"""CPU: the argument checks of the operators that shape scores, share prefixes or stand between blocks.  Nothing is launched."""
import re
import struct
from pathlib import Path

import pytest
import torch

from nanopd_b200 import _lib, decoder_step, norms, paged_kernels

NULL = None


def scored(**kw):
    a = dict(scale=0.1, cap=5.0, slopes=NULL, window=0, S=1, hq=4, hkv=2, d=128, bs=16, blk=4, nb=8, stride=2 * 16 * 128, dtype=_lib.NPD_DTYPE_F16,
             flags=0)
    a.update(kw)
    return _lib.load().npd_paged_scored_attention(NULL, NULL, NULL, NULL, NULL, NULL, a["scale"], a["cap"], a["slopes"], a["window"], a["S"], a["hq"],
                                                  a["hkv"], a["d"], a["bs"], a["blk"], a["nb"], a["stride"], a["blk"], a["dtype"], NULL, 0, NULL,
                                                  a["flags"], NULL)


def prefill(**kw):
    a = dict(scale=0.1, cap=5.0, window=0, chunks=1, hq=4, hkv=2, d=128, bs=16, dtype=_lib.NPD_DTYPE_BF16, flags=0)
    a.update(kw)
    return _lib.load().npd_paged_scored_prefill_attention(NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, a["chunks"], a["scale"], a["cap"], NULL,
                                                          a["window"], a["hq"], a["hkv"], a["d"], a["bs"], 4, 8, 4096, 4, a["dtype"], NULL, 0, NULL,
                                                          a["flags"], NULL)


def shared(**kw):
    a = dict(scale=0.1, S=2, groups=1, hq=4, hkv=2, d=128, bs=16, dtype=_lib.NPD_DTYPE_F16, flags=0)
    a.update(kw)
    return _lib.load().npd_paged_shared_prefix_attention(NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, a["scale"], a["S"], a["groups"], a["hq"],
                                                         a["hkv"], a["d"], a["bs"], 4, 8, 4096, 4, a["dtype"], NULL, 0, NULL, a["flags"], NULL)


@pytest.mark.parametrize("call,kw,code,match", [
    (scored, dict(cap=-1.0), _lib.NPD_ERR_INVALID_ARG, b"cap"), (scored, dict(cap=float("nan")), _lib.NPD_ERR_INVALID_ARG, b"cap"),
    (scored, dict(cap=1e-35), _lib.NPD_ERR_INVALID_ARG, b"cap"), (scored, dict(cap=float("inf")), _lib.NPD_ERR_INVALID_ARG, b"cap"),
    (scored, dict(window=-1), _lib.NPD_ERR_INVALID_ARG, b"window"), (scored, dict(slopes=2), _lib.NPD_ERR_INVALID_ARG, b"slopes"),
    (scored, dict(scale=-0.5), _lib.NPD_ERR_INVALID_ARG, b"scale"), (scored, dict(scale=float("inf")), _lib.NPD_ERR_INVALID_ARG, b"scale"),
    (scored, dict(flags=2), _lib.NPD_ERR_INVALID_ARG, b"MAX_CTAS"), (scored, dict(d=96), _lib.NPD_ERR_UNSUPPORTED, b"head_dim"),
    (scored, dict(bs=12), _lib.NPD_ERR_UNSUPPORTED, b"block_size"), (scored, dict(dtype=2), _lib.NPD_ERR_UNSUPPORTED, b"float16"),
    (scored, dict(hq=5), _lib.NPD_ERR_INVALID_ARG, b"multiple"), (scored, dict(), _lib.NPD_ERR_INVALID_ARG, b"NULL"),
    (scored, dict(S=0), _lib.NPD_OK, None),
    (prefill, dict(cap=-1.0), _lib.NPD_ERR_INVALID_ARG, b"cap"), (prefill, dict(window=-3), _lib.NPD_ERR_INVALID_ARG, b"window"),
    (prefill, dict(scale=float("nan")), _lib.NPD_ERR_INVALID_ARG, b"scale"), (prefill, dict(flags=1), _lib.NPD_ERR_INVALID_ARG, b"MAX_CTAS"),
    (prefill, dict(d=32), _lib.NPD_ERR_UNSUPPORTED, b"head_dim"), (prefill, dict(hq=258), _lib.NPD_ERR_UNSUPPORTED, b"128 q heads"),
    (prefill, dict(), _lib.NPD_ERR_INVALID_ARG, b"NULL"), (prefill, dict(chunks=0), _lib.NPD_OK, None),
    (shared, dict(groups=0), _lib.NPD_ERR_INVALID_ARG, b"groups"), (shared, dict(groups=4097), _lib.NPD_ERR_INVALID_ARG, b"groups"),
    (shared, dict(scale=-1.0), _lib.NPD_ERR_INVALID_ARG, b"scale"), (shared, dict(flags=4), _lib.NPD_ERR_INVALID_ARG, b"MAX_CTAS"),
    (shared, dict(), _lib.NPD_ERR_INVALID_ARG, b"NULL"), (shared, dict(d=80), _lib.NPD_ERR_UNSUPPORTED, b"head_dim"),
])
def test_entry_points_refuse_before_any_launch(call, kw, code, match):
    assert call(**kw) == code
    if match:
        assert match in _lib.load().npd_last_error()


def test_residual_norms_entry_point_refuses():
    f = _lib.load().npd_residual_norms
    args = lambda rows=4, hidden=64, dtype=1, stride=64: (NULL,) * 7 + (1.0, 1e-6, 0.0, rows, hidden, stride, 64, 0, 64, 64, dtype, NULL)  # noqa: E731
    assert f(*args(hidden=60)) == _lib.NPD_ERR_UNSUPPORTED and f(*args(hidden=32776)) == _lib.NPD_ERR_UNSUPPORTED
    assert f(*args(dtype=7)) == _lib.NPD_ERR_UNSUPPORTED and f(*args(rows=-1)) == _lib.NPD_ERR_INVALID_ARG
    assert f(*args(rows=0)) == _lib.NPD_OK and f(*args()) == _lib.NPD_ERR_INVALID_ARG
    p = 1 << 20
    bad = lambda **kw: f(*[{**dict(enumerate((p, 2 * p, 3 * p, 4 * p, 5 * p, NULL, NULL, 1.0, 1e-6, 0.0, 4, 64, 64, 64, 0, 64, 64, 1, NULL))),  # noqa: E731
                            **{int(k[1:]): v for k, v in kw.items()}}[i] for i in range(19)])
    for kw in (dict(a2=p + 2), dict(a12=60), dict(a13=68), dict(a6=6 * p, a14=32), dict(a4=p + 8)):
        assert bad(**kw) == _lib.NPD_ERR_INVALID_ARG


def test_packed_calls_carry_the_entry_points_arguments():
    """Every packing has the device and then one 8-byte slot for each argument of its entry point; floats sit where floats go."""
    from ctypes import c_float
    for name, pack in (("npd_paged_scored_attention", paged_kernels._pack_scored), ("npd_paged_scored_prefill_attention", paged_kernels._pack_scored_prefill),
                       ("npd_paged_shared_prefix_attention", paged_kernels._pack_shared), ("npd_residual_norms", norms._pack)):
        types = _lib.SIGNATURES[name][1]
        fmt = pack.__self__.format
        fields = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qQd])", fmt))
        assert fields[0] == "q" and len(fields) == 1 + len(types) and struct.calcsize(fmt) == 8 * len(fields), name
        assert [c == "d" for c in fields[1:]] == [t is c_float for t in types], name
    lib = _lib.load()
    assert lib.npd_call_packed(_lib.NPD_OP_RESIDUAL_NORMS, None) == _lib.NPD_ERR_INVALID_ARG


def test_workspace_of_the_shared_prefix_operator():
    f = _lib.load().npd_shared_prefix_workspace_bytes
    assert f(2, 0, 0, 2, 128, 0) == 0 and f(-1, 1, 4, 2, 128, 0) == 0
    assert 0 < f(1, 1, 4, 2, 64, 0) < f(256, 1, 32, 8, 128, 0) < f(4096, 4096, 32, 8, 128, 0) < 1 << 30


def test_python_operators_refuse_cpu_tensors():
    q, kc, bt, sl = torch.zeros(2, 4, 64), torch.zeros(4, 2, 16, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kernels.paged_scored_attention(q, q, kc, kc, bt, sl, 0.1, 16, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kernels.paged_shared_prefix_attention(q, q, kc, kc, bt, sl, sl, sl[:1], 0.1, 16, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kernels.paged_scored_prefill_attention(q, q, kc, kc, bt, [0], [1], [0], 0.1, 16, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        norms.residual_norms(torch.zeros(2, 64), torch.zeros(2, 64), torch.zeros(64))
    with pytest.raises(RuntimeError, match="tensors"):
        norms.residual_norms(None, None, None)
    with pytest.raises(RuntimeError, match="tensors"):
        paged_kernels.paged_scored_prefill_attention(q, q, kc, kc, bt, [0.5], [1], [0], 0.1, 16, 2)


def test_rows_apart():
    """Rows of 64 bytes: one behind the other, columns of one buffer, and what overlaps."""
    apart = norms._apart
    assert apart(0, 640, 64, 640, 640, 64, 64) and not apart(0, 640, 64, 576, 640, 64, 64)
    assert apart(0, 1984, 192, 64, 1984, 192, 64) and apart(128, 1984, 192, 0, 1984, 192, 64)
    assert not apart(0, 1984, 192, 32, 1984, 192, 64) and not apart(0, 1984, 192, 64, 1984, 256, 64) and not apart(0, 640, 64, 0, 640, 64, 64)


def test_decoder_shapes():
    plain = decoder_step.DecoderShape()
    assert not plain.fused_norms and plain.score_cap == 0 and plain.window == 0
    assert decoder_step.DecoderShape(post_norms=True).fused_norms and decoder_step.DecoderShape(residual_scale=0.5).fused_norms
    assert decoder_step.DecoderShape(post_norms=True).param_count == plain.param_count + 2 * plain.num_layers * plain.hidden


def test_cap_polynomial_of_the_prompt_kernel():
    """The coefficients in the source against tanh: within 2.2e-6 relative over the range that they serve."""
    src = (Path(__file__).resolve().parents[1] / "nanopd_b200" / "csrc" / "prefill_kernel.cuh").read_text()
    fit = [float(x) for x in re.search(r"fit\[4\] = \{([^}]*)\}", src).group(1).split(",")]
    z = torch.linspace(-0.6, 0.6, 20001, dtype=torch.float64)
    z = z[z != 0]
    p = sum(c * z ** (2 * k + 1) for k, c in enumerate(fit))
    assert float(((p - torch.tanh(z)) / torch.tanh(z)).abs().max()) < 2.2e-6
