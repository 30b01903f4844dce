"""GPU: the norms, gate and residual sum between two blocks against a plain form in 64 bits."""
import pytest
import torch

from nanopd_b200 import norms
from oracle import shaped_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def make(T, H, dtype, post=True, gate=None, seed=0, gain=2.0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    return dict(x=(r(T, H) * 0.7).to(dtype), residual=(r(T, H) * gain).to(dtype), weight=(1 + 0.2 * r(H)).to(dtype),
                post_weight=(1 + 0.2 * r(H)).to(dtype) if post else None,
                gate={None: None, "channel": (0.5 * r(H)).to(dtype), "token": (0.5 * r(T, H)).to(dtype)}[gate])


def expect(got, a, **kw):
    """Half a step of the type for each output's rounding; in front of it 32-bit arithmetic: the mean of H squares is a tree
    of at most 8 values in a row, 5 shuffles and 16 warps (fewer than 64 additions, each 2^-24), then a product, a root
    (2 units) and three products — below 80 * 2^-24 relative on a normed value, and on the sum's terms the same."""
    r, h, terms = shaped_oracle.residual_norms(**a, **kw)
    half, f32 = torch.finfo(a["x"].dtype).eps / 2, 80 * 2.0 ** -24
    tiny = torch.finfo(a["x"].dtype).smallest_normal * torch.finfo(a["x"].dtype).eps      # steps of subnormal results
    tol_r = half * r.abs() + f32 * terms + tiny
    # an error of the sum reaches its norm scaled by the norm's factor; the mean moves by less than the largest term's error
    factor = (h.abs() + 1e-30) / (r.abs() + 1e-30)
    tol_h = half * h.abs() + f32 * (h.abs() + 3 * factor * terms) + tiny
    for name, x, want, tol in (("residual", got[0], r, tol_r), ("normed", got[1], h, tol_h)):
        assert torch.isfinite(x).all(), name
        off = (x.double() - want).abs()
        assert (off <= tol).all(), f"{name}: {float((off / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H", [(1, 8), (1, 4096), (3, 64), (5, 248), (7, 264), (4, 1024), (257, 1536), (33, 4104), (2, 8192), (3, 16384), (2, 32768), (9, 512)])
@pytest.mark.parametrize("post,gate", [(True, None), (False, None), (True, "channel"), (False, "token")])
def test_shapes(dtype, T, H, post, gate):
    a = make(T, H, dtype, post, gate)
    expect(norms.residual_norms(**a), a)
    expect(norms.residual_norms(**a, residual_scale=0.22, eps=1e-5, weight_offset=1.0), a, residual_scale=0.22, eps=1e-5, weight_offset=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_and_strided_rows(dtype):
    T, H = 37, 1536
    a = make(T, H, dtype)
    want = norms.residual_norms(**a)
    wide = torch.full((T, 3 * H + 64), 5.0, dtype=dtype, device=DEV)
    wide[:, :H], wide[:, H + 32:2 * H + 32] = a["x"], a["residual"]
    x, res = wide[:, :H], wide[:, H + 32:2 * H + 32]
    got = norms.residual_norms(x, res, a["weight"], a["post_weight"], residual_out=res, out=x)
    assert got[0] is res and got[1] is x
    assert torch.equal(x, want[1]) and torch.equal(res, want[0])
    assert (wide[:, H:H + 32] == 5).all() and (wide[:, 2 * H + 32:] == 5).all()
    # the other way round: the norm over the residual, the sum over the block's output
    b = make(T, H, dtype)
    got = norms.residual_norms(b["x"], b["residual"], b["weight"], b["post_weight"], residual_out=b["x"], out=b["residual"])
    assert torch.equal(b["x"], want[0]) and torch.equal(b["residual"], want[1])


def test_rows_behind_the_last_are_left_alone():
    a = make(5, 256, torch.bfloat16)
    ro, o = (torch.full((8, 256), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    norms.residual_norms(**a, residual_out=ro[:5], out=o[:5])
    assert (ro[5:] == 3).all() and (o[5:] == 3).all()


def test_gates_expanded_and_of_one_row():
    a = make(6, 512, torch.bfloat16, gate="channel")
    want = norms.residual_norms(**a)
    b = dict(a, gate=a["gate"].expand(6, 512))
    assert all(torch.equal(x, y) for x, y in zip(norms.residual_norms(**b), want))
    one = {k: (v[:1] if v is not None and v.dim() == 2 else v) for k, v in a.items()}
    one["gate"] = a["gate"][None]
    assert torch.equal(norms.residual_norms(**one)[0], want[0][:1])


def test_zero_rows_zero_values_and_infinities():
    a = make(0, 256, torch.float16)
    r, h = norms.residual_norms(**a)
    assert r.shape == h.shape == (0, 256)
    a = make(3, 256, torch.float16)
    a["x"].zero_(), a["residual"].zero_()
    r, h = norms.residual_norms(**a)
    assert (r == 0).all() and (h == 0).all()
    a = make(3, 256, torch.float16)
    a["residual"][1, 7] = float("inf")
    r, h = norms.residual_norms(**a)
    good = make(3, 256, torch.float16)
    want = norms.residual_norms(**good)
    assert torch.equal(r[[0, 2]], want[0][[0, 2]]) and torch.equal(h[[0, 2]], want[1][[0, 2]])
    assert torch.isinf(r[1, 7]) and torch.isnan(h[1, 7])


def test_sums_beyond_a_half_types_range():
    """Values whose squares pass the 16-bit range: the norms are in 32 bits."""
    a = make(4, 4096, torch.float16, gain=900.0)
    a["x"] *= 500
    expect(norms.residual_norms(**a), a)


def test_graph_and_side_stream():
    a = make(64, 4096, torch.bfloat16)
    want = norms.residual_norms(**a)
    ro, o = torch.empty_like(a["x"]), torch.empty_like(a["x"])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norms.residual_norms(**a, residual_out=ro, out=o)
    ro.zero_(), o.zero_()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        g.replay()
        torch.cuda.current_stream().synchronize()
    assert torch.equal(ro, want[0]) and torch.equal(o, want[1])


def test_refusals():
    a = make(4, 256, torch.bfloat16)
    call = lambda **kw: norms.residual_norms(**{**a, **kw})  # noqa: E731
    bad = [dict(x=a["x"].cpu()), dict(x=a["x"][:, :250]), dict(x=a["x"].double()), dict(residual=a["residual"].float()), dict(residual=a["residual"][:3]),
           dict(weight=a["weight"][:-8]), dict(weight=a["weight"].float()), dict(post_weight=a["weight"][None]), dict(gate=a["x"][:2]),
           dict(gate=a["x"][:, ::2]), dict(x=a["x"].t().contiguous().t()), dict(out=a["x"].clone()[:, :128]), dict(x=None),
           dict(residual_out=a["weight"]), dict(weight=a["weight"].cpu())]
    for kw in bad:
        with pytest.raises(RuntimeError):
            call(**kw)
    both = torch.empty(5, 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="overlaps"):
        call(residual_out=both[:4], out=both[1:])
    with pytest.raises(RuntimeError, match="overlaps"):
        call(x=both[:4], out=both[1:])
    with pytest.raises(RuntimeError, match="overlaps"):
        call(gate=both[:4], out=both[:4])
    with pytest.raises(RuntimeError, match="aligned"):
        flat = torch.empty(4 * 256 + 8, dtype=torch.bfloat16, device=DEV)
        call(x=flat[1:1 + 4 * 256].view(4, 256))
    with pytest.raises(RuntimeError, match="strides"):
        call(x=torch.empty(4, 260, dtype=torch.bfloat16, device=DEV)[:, :256])
