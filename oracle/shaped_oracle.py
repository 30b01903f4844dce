"""Plain 64-bit forms of the operators that shape scores or stand between blocks (test infrastructure only).

Every attention form returns, beside its rows, what a tolerance is built from: ``A = sum_j p_j |v_j|`` (an error of a
relative size d in every probability moves a row by at most 2 d A) and the softmax sum relative to the row's maximum.
"""
from __future__ import annotations

import math

import torch


def gather_pages(cache: torch.Tensor, table_row: torch.Tensor, lo: int, hi: int) -> torch.Tensor:
    """Tokens [lo, hi) of a sequence, [Hkv, hi - lo, D] in 64 bits.  Pages wholly before ``lo`` are not looked up."""
    bs = cache.size(2)
    first = lo // bs
    pages = table_row[first:(hi + bs - 1) // bs].long()
    rows = cache[pages].permute(1, 0, 2, 3).reshape(cache.size(1), -1, cache.size(3))
    return rows[:, lo - first * bs:hi - first * bs].double()


def shaped_scores(q, k, scale, cap, slopes, q_pos, k_pos):
    """q [H, n, D] of one kv head's group, k [m, D]; positions of queries and keys.  [H, n, m]"""
    x = torch.einsum("hnd,md->hnm", q.double(), k) * scale
    if cap:
        x = cap * torch.tanh(x / cap)
    if slopes is not None:
        x = x - slopes.double()[:, None, None] * (q_pos[:, None] - k_pos[None, :]).double()
    return x


def attend(q, k_cache, v_cache, table_row, start, scale, cap=0.0, slopes=None, window=0):
    """Causal attention of queries q [n, Hq, D] at positions start .. start + n - 1 over the pages of one table row.
    Returns (out [n, Hq, D], A [n, Hq, D], l [n, Hq])."""
    n, hq, d = q.shape
    hkv = k_cache.size(1)
    G = hq // hkv
    dev = q.device
    lo, hi = (max(0, start - window + 1) if window else 0), start + n
    q_pos, k_pos = torch.arange(start, hi, device=dev), torch.arange(lo, hi, device=dev)
    hidden = k_pos[None, :] > q_pos[:, None]
    if window:
        hidden |= k_pos[None, :] <= q_pos[:, None] - window
    k, v = gather_pages(k_cache, table_row, lo, hi), gather_pages(v_cache, table_row, lo, hi)
    out = torch.empty(n, hq, d, dtype=torch.float64, device=dev)
    A = torch.empty_like(out)
    l = torch.empty(n, hq, dtype=torch.float64, device=dev)
    for h in range(hkv):
        sl = slice(h * G, (h + 1) * G)
        x = shaped_scores(q[:, sl].permute(1, 0, 2), k[h], scale, cap, None if slopes is None else slopes[sl], q_pos, k_pos)
        x = x.masked_fill(hidden, -math.inf)
        e = (x - x.amax(-1, keepdim=True)).exp()
        s = e.sum(-1, keepdim=True)
        pr = e / s
        out[:, sl] = torch.einsum("hnm,md->nhd", pr, v[h])
        A[:, sl] = torch.einsum("hnm,md->nhd", pr, v[h].abs())
        l[:, sl] = s[..., 0].T
    return out, A, l


def attend_single(q, k_cache, v_cache, block_tables, seq_lens, scale, cap=0.0, slopes=None, window=0):
    """One query token per sequence; a sequence of length 0 gets a zero row."""
    S, hq, d = q.shape
    out = torch.zeros(S, hq, d, dtype=torch.float64, device=q.device)
    A, l = torch.zeros_like(out), torch.ones(S, hq, dtype=torch.float64, device=q.device)
    for s, n in enumerate(seq_lens.tolist()):
        if n > 0:
            o, a, ll = attend(q[s:s + 1], k_cache, v_cache, block_tables[s], n - 1, scale, cap, slopes, window)
            out[s], A[s], l[s] = o[0], a[0], ll[0]
    return out, A, l


def attention_tolerance(out, A, l, keys: int, dtype, v_max: float):
    """How far a kernel's row may be from ``out``, element by element:
    * the probabilities are rounded to the 16-bit type before the product with V (half a step each: A * eps / 2), and the
      result once more (|out| * eps / 2);
    * a probability below the type's smallest normal number is off by at most half of its smallest subnormal step
      (fp16; the row sum is at least l relative to the largest probability, which is stored as 1 or more);
    * the exponent's error: scores and their shaping in 32 bits (products of 16-bit values are exact, sums of up to 256 of
      them and the tanh stay below 3e-5 for scores of up to 60), and 7.5e-5 of the cubic 2^f of the prompt kernel.
      Together below d = 1.5e-4, which moves a row by at most 2 d A."""
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return half * (A + out.abs()) * 1.01 + 2 * 1.5e-4 * A + (keys * tiny * v_max / l.clamp(min=1.0))[..., None] + 1e-7


def residual_norms(x, residual, weight, post_weight=None, gate=None, residual_scale=1.0, eps=1e-6, weight_offset=0.0):
    """(residual_out, out, |terms of the sum|) in 64 bits."""
    f = lambda t: None if t is None else t.double()  # noqa: E731
    x, residual, weight, post_weight, gate = map(f, (x, residual, weight, post_weight, gate))
    y = x
    if post_weight is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (post_weight + weight_offset)
    if gate is not None:
        y = gate * y
    y = residual_scale * y
    r = residual + y
    out = r / (r.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (weight + weight_offset)
    return r, out, residual.abs() + y.abs()
