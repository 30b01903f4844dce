"""The operators whose speed this repository watches, each with a plain form in elementary torch operations.

Four operators of one serving path over the paged cache (head counts, head sizes and block sizes are those of the
repository's own configurations and of shapes that its kernels take):

* ``decode``: one query token per sequence over paged keys and values, with scores capped by a tanh, a bias that is
  linear in the distance to the key, and a sliding window (each of them optional);
* ``prompt``: the same scores for chunks of prompts, causal;
* ``shared``: one query token per sequence for a batch whose sequences share the first pages of their tables;
* ``norms``: what stands between two blocks of a layer: the norm of a block's output, its gate and scale, the residual
  sum, and the norm that feeds the next block.

A case is a dict of plain values; its lengths follow from the case alone (``lens_seed``), its values from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a single user's chat: latency of one launch is all there is
        dict(name="decode one sequence", op="decode", dtype="bf16", hq=32, hkv=8, d=128, block=16, seqs=1, lo=700, hi=700, skew=0.0,
             cap=50.0, slopes=False, window=0, lens_seed=1),
        # a full decode batch with the ragged contexts of the main decode workload, every layer's scores capped
        dict(name="decode full batch", op="decode", dtype="bf16", hq=32, hkv=8, d=128, block=16, seqs=256, lo=32, hi=8192, skew=0.8,
             cap=50.0, slopes=False, window=0, lens_seed=2),
        # long contexts through a layer that only looks back 1024 tokens, with a distance bias
        dict(name="decode window bias", op="decode", dtype="fp16", hq=12, hkv=2, d=128, block=16, seqs=61, lo=900, hi=9000, skew=0.0,
             cap=0.0, slopes=True, window=1024, lens_seed=3),
        # a short follow-up question behind a cached conversation
        dict(name="prompt short", op="prompt", dtype="fp16", hq=12, hkv=2, d=128, block=16, prompts=2, lo=23, hi=77, chunk=0, start=205,
             cap=0.0, slopes=True, window=0, lens_seed=4),
        # one scheduler step with the 512-token chunks of four prompts
        dict(name="prompt chunks", op="prompt", dtype="bf16", hq=32, hkv=8, d=128, block=16, prompts=4, lo=1024, hi=4096, chunk=512, start=0,
             cap=50.0, slopes=False, window=0, lens_seed=5),
        # a document in one piece, a layer with capped scores and a sliding window
        dict(name="prompt long window", op="prompt", dtype="bf16", hq=32, hkv=8, d=128, block=16, prompts=1, lo=8111, hi=8111, chunk=0, start=0,
             cap=30.0, slopes=False, window=4096, lens_seed=6),
        # a handful of requests behind one system prompt
        dict(name="shared small batch", op="shared", dtype="fp16", hq=12, hkv=2, d=128, block=16, groups=1, seqs=16, prefix_lo=1000, prefix_hi=1000,
             lo=5, hi=300, lens_seed=7),
        # many requests about the same long document
        dict(name="shared long prefix", op="shared", dtype="bf16", hq=32, hkv=8, d=128, block=16, groups=1, seqs=256, prefix_lo=8192, prefix_hi=8192,
             lo=32, hi=700, lens_seed=8),
        # several applications on one server, each with its own instructions and examples
        dict(name="shared eight prefixes", op="shared", dtype="bf16", hq=32, hkv=8, d=128, block=16, groups=8, seqs=133, prefix_lo=700, prefix_hi=4000,
             lo=16, hi=1100, lens_seed=9),
        # between two blocks of a layer, a single token
        dict(name="norms one token", op="norms", dtype="bf16", tokens=1, hidden=4096, post=True, gate="none", scale=1.0, offset=1.0),
        # a decode batch of a smaller model, the block's output scaled per channel
        dict(name="norms batch gate", op="norms", dtype="fp16", tokens=257, hidden=1536, post=False, gate="channel", scale=0.22, offset=0.0),
        # the prompt tokens of one step
        dict(name="norms prompt", op="norms", dtype="bf16", tokens=8191, hidden=4096, post=True, gate="none", scale=1.0, offset=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8, 128), (12, 2, 128), (16, 16, 64), (14, 2, 64), (16, 2, 256), (24, 8, 128)]


def draw(rng):
    op = rng.choice(["decode", "prompt", "shared", "norms"])
    dtype = rng.choice(["bf16", "fp16"])
    seed = rng.randrange(1 << 30)
    if op == "norms":
        post = rng.random() < 0.5
        gate = rng.choice(["none", "channel", "token"])
        hidden = 8 * _log(rng, 8, 1024)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        most = min(8191, (3 << 24) // _SIZE[dtype] // hidden)
        return dict(op=op, dtype=dtype, tokens=_log(rng, 1, max(1, most)), hidden=hidden, post=post, gate=gate,
                    scale=rng.choice([1.0, 0.22, 0.5]), offset=rng.choice([0.0, 1.0]))
    hq, hkv, d = rng.choice(_HEADS)
    block = rng.choice([8, 16, 16, 32])
    if op == "shared":
        seqs = _log(rng, 2, 220)
        prefix = _log(rng, 64, 8000 if seqs * hkv * d <= 220 * 1024 else 3000)
        return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, block=block, groups=min(seqs, _log(rng, 1, 12)), seqs=seqs, prefix_lo=max(1, prefix // 2),
                    prefix_hi=prefix, lo=1, hi=_log(rng, 2, 700), lens_seed=seed)
    cap = rng.choice([0.0, 30.0, 50.0])
    slopes = rng.random() < (0.4 if cap else 0.7)
    window = rng.choice([0, _log(rng, 16, 4096)])
    if op == "decode":
        seqs = _log(rng, 1, 200)
        hi = _log(rng, 16, min(16000, 600_000 // seqs))
        return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, block=block, seqs=seqs, lo=1, hi=hi, skew=rng.choice([0.0, 0.8]), cap=cap, slopes=slopes,
                    window=window, lens_seed=seed)
    hi = _log(rng, 16, 5000)
    return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, block=block, prompts=rng.randint(1, max(1, min(4, 8000 // hi))), lo=max(1, hi // 3), hi=hi,
                chunk=rng.choice([0, 512]), start=rng.choice([0, _log(rng, 1, 1500)]), cap=cap, slopes=slopes, window=window, lens_seed=seed)


# ---------------------------------------------------------------------------------------------------------------
# lengths and work, from the case alone
# ---------------------------------------------------------------------------------------------------------------
def _lens(c):
    """Tokens of each sequence, the query's own token included."""
    r = random.Random(c["lens_seed"])
    if c["skew"] > 0:
        mid = math.sqrt(c["lo"] * c["hi"])
        mid = max(mid, c["hi"] / 8)
        return [int(min(c["hi"], max(c["lo"], round(mid * math.exp(r.gauss(0.0, c["skew"])))))) for _ in range(c["seqs"])]
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]


def _chunks(c):
    """(prompt, first position, tokens) of each chunk; and the tokens of each prompt with what was cached before it."""
    r = random.Random(c["lens_seed"])
    found, ends = [], []
    for i in range(c["prompts"]):
        n = r.randint(c["lo"], c["hi"])
        step = c["chunk"] or n
        found += [(i, c["start"] + at, min(step, n - at)) for at in range(0, n, step)]
        ends.append(c["start"] + n)
    return found, ends


def _groups(c):
    """(sequences, tokens of the shared prefix) of each group, and each sequence's own tokens behind it."""
    r = random.Random(c["lens_seed"])
    cuts = sorted(r.sample(range(1, c["seqs"]), c["groups"] - 1)) if c["groups"] > 1 else []
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [c["seqs"]])]
    groups = [(n, r.randint(c["prefix_lo"], c["prefix_hi"]) // c["block"] * c["block"]) for n in sizes]
    return groups, [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]


def work(c):
    e = _SIZE[c["dtype"]]
    if c["op"] == "norms":
        rows = c["tokens"] * c["hidden"]
        gate = {"none": 0, "channel": c["hidden"], "token": rows}[c["gate"]]
        return {"bytes": e * (4 * rows + gate + (2 if c["post"] else 1) * c["hidden"]), "flops": 10 * rows}
    row, kv = c["hq"] * c["d"] * e, 2 * c["hkv"] * c["d"] * e
    if c["op"] == "decode":
        seen = [min(n, c["window"]) if c["window"] else n for n in _lens(c)]
        tokens, pairs, queries = sum(seen), sum(seen), c["seqs"]
        index = 4 * sum(-(-n // c["block"]) for n in seen) + 4 * c["seqs"]
    elif c["op"] == "prompt":
        found, ends = _chunks(c)
        w = c["window"] or 1 << 60
        first = {i: max(0, min(s for j, s, _ in found if j == i) - w + 1) for i in range(c["prompts"])}
        tokens = sum(e2 - first[i] for i, e2 in enumerate(ends))
        queries = sum(n for _, _, n in found)
        pairs = sum(int(np.minimum(np.arange(s + 1, s + n + 1), w).sum()) for _, s, n in found)
        index = 4 * tokens // c["block"]
    else:
        groups, tails = _groups(c)
        shared = [p for n, p in groups for _ in range(n)]
        tokens = sum(p for _, p in groups) + sum(tails)
        pairs, queries = sum(shared) + sum(tails), c["seqs"]
        index = 4 * tokens // c["block"] + 4 * c["seqs"]
    return {"bytes": tokens * kv + 2 * queries * row + index, "flops": 4 * c["hq"] * c["d"] * pairs}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _slopes(hq, device):
    """The usual geometric ladder of slopes, one for each query head."""
    return torch.exp2(-8.0 * torch.arange(1, hq + 1, dtype=torch.float32, device=device) / hq)


def _tables(rows, total, gen, device):
    """Block tables of a pool whose pages lie in random order: ``rows`` holds, for each table row, the page numbers counted
    in the order in which they were handed out."""
    perm = torch.randperm(total, generator=gen, device=device).to(torch.int32)
    width = max(1, max(len(r) for r in rows))
    at = np.zeros((len(rows), width), dtype=np.int64)
    for i, r in enumerate(rows):
        at[i, :len(r)] = r
    return perm[torch.from_numpy(at).to(device)].contiguous()


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dt = _DTYPE[c["dtype"]]

    def randn(*shape, gain=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * gain).to(dt)

    s = dict(c)
    if c["op"] == "norms":
        T, H = c["tokens"], c["hidden"]
        s["x"], s["residual"] = randn(T, H, gain=0.7), randn(T, H, gain=4.0)
        s["weight"] = randn(H, gain=0.2) + (1.0 - c["offset"])
        s["post_weight"] = randn(H, gain=0.2) + (1.0 - c["offset"]) if c["post"] else None
        s["gate"] = {"none": lambda: None, "channel": lambda: randn(H, gain=0.5), "token": lambda: randn(T, H, gain=0.5)}[c["gate"]]()
        s["residual_out"], s["out"] = torch.empty_like(s["residual"]), torch.empty_like(s["x"])
        return s
    hq, hkv, d, block = c["hq"], c["hkv"], c["d"], c["block"]
    if c["op"] == "decode":
        lens = _lens(c)
        rows, total = [], 0
        for n in lens:
            pages = -(-n // block)
            rows.append(range(total, total + pages))
            total += pages
        queries = c["seqs"]
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    elif c["op"] == "prompt":
        found, ends = _chunks(c)
        pages, total = [], 0
        for n in ends:
            pages.append(range(total, total + -(-n // block)))
            total += -(-n // block)
        rows = [pages[i] for i, _, _ in found]
        s["starts"], s["tokens"] = [a for _, a, _ in found], [n for _, _, n in found]
        s["offsets"] = [int(v) for v in np.cumsum([0] + s["tokens"][:-1])]
        queries = sum(s["tokens"])
        s["starts_dev"], s["tokens_dev"], s["offsets_dev"] = (torch.tensor(s[k], dtype=torch.int64, device=dev) for k in ("starts", "tokens", "offsets"))
    else:
        groups, tails = _groups(c)
        rows, lens, total = [], [], 0
        for n, p in groups:
            head = list(range(total, total + p // block))
            total += len(head)
            for _ in range(n):
                own_pages = -(-tails[len(rows)] // block)
                lens.append(p + tails[len(rows)])
                rows.append(head + list(range(total, total + own_pages)))
                total += own_pages
        queries = c["seqs"]
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["group_offsets"] = torch.tensor(np.cumsum([0] + [n for n, _ in groups]), dtype=torch.int32, device=dev)
        s["shared_lens"] = torch.tensor([p for _, p in groups], dtype=torch.int32, device=dev)
    s["block_tables"] = _tables(rows, total, gen, dev)
    # models that cap their scores do it because the scores get large
    s["query"] = randn(queries, hq, d, gain=4.0 if c.get("cap") else 1.0)
    s["k_cache"], s["v_cache"] = randn(total, hkv, block, d), randn(total, hkv, block, d)
    s["scale"] = float(d) ** -0.5
    s["slope"] = _slopes(hq, dev) if c.get("slopes") else None
    s["out"] = torch.empty_like(s["query"])
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _gathered(cache, tables):
    """[rows, kv heads, tokens, d] in 32 bits: the pages of each table row, one after another."""
    r, n = tables.shape
    _, hkv, block, d = cache.shape
    return cache[tables.long()].permute(0, 2, 1, 3, 4).reshape(r, hkv, n * block, d).float()


def _attend(q, k, v, positions, last, s):
    """q [R, n, Hq, D] at ``positions`` [R, n], k and v [R, Hkv, L, D]: key j of row r is there for j <= ``last`` [R, n]."""
    R, n, hq, d = q.shape
    hkv, L = k.shape[1], k.shape[2]
    q = q.float().reshape(R, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(R, hkv, (hq // hkv) * n, d)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(R, hkv, hq // hkv, n, L)
    if s.get("cap"):
        x = x.div_(s["cap"]).tanh_().mul_(s["cap"])
    away = positions[:, :, None] - torch.arange(L, device=q.device)[None, None, :]
    if s.get("slope") is not None:
        x = x - s["slope"].view(1, hkv, hq // hkv, 1, 1) * away.float()[:, None, None]
    hidden = away < (positions - last)[:, :, None]
    if s.get("window"):
        hidden = hidden | (away >= s["window"])
    x = x.masked_fill_(hidden[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    x = x.div_(x.sum(-1, keepdim=True)).view(R, hkv, (hq // hkv) * n, L)
    return torch.matmul(x, v).view(R, hkv, hq // hkv, n, d).permute(0, 3, 1, 2, 4).reshape(R, n, hq, d)


def _plain_single(s):
    k, v = _gathered(s["k_cache"], s["block_tables"]), _gathered(s["v_cache"], s["block_tables"])
    at = (s["seq_lens"].long() - 1)[:, None]
    return _attend(s["query"][:, None], k, v, at, at, s)[:, 0].to(s["query"].dtype)


def _plain_prompt(s):
    widest = max(s["tokens"])
    k, v = _gathered(s["k_cache"], s["block_tables"]), _gathered(s["v_cache"], s["block_tables"])
    inside = torch.arange(widest, device=k.device)[None].minimum(s["tokens_dev"][:, None] - 1)
    rows = s["offsets_dev"][:, None] + inside
    at = s["starts_dev"][:, None] + inside
    o = _attend(s["query"][rows], k, v, at, at, s)
    packed = torch.arange(s["query"].shape[0], device=k.device)
    chunk = torch.searchsorted(s["offsets_dev"], packed, right=True) - 1
    return o[chunk, packed - s["offsets_dev"][chunk]].to(s["query"].dtype)


def _plain_norms(s):
    dt = s["x"].dtype

    def norm(t, w):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * (w.float() + s["offset"])

    y = s["x"].float()
    if s["post_weight"] is not None:
        y = norm(y, s["post_weight"])
    if s["gate"] is not None:
        y = y * s["gate"].float()
    r = s["residual"].float() + s["scale"] * y
    return {"residual": r.to(dt), "normed": norm(r, s["weight"]).to(dt)}


def run(s):
    if not own:
        return {"decode": _plain_single, "shared": _plain_single, "prompt": _plain_prompt, "norms": _plain_norms}[s["op"]](s)
    from nanopd_b200 import norms, paged_kernels
    if s["op"] == "norms":
        r, h = norms.residual_norms(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], residual_scale=s["scale"], eps=1e-6,
                                    weight_offset=s["offset"], residual_out=s["residual_out"], out=s["out"])
        return {"residual": r, "normed": h}
    a = (s["out"], s["query"], s["k_cache"], s["v_cache"], s["block_tables"])
    width = s["block_tables"].shape[1]
    if s["op"] == "decode":
        paged_kernels.paged_scored_attention(*a, s["seq_lens"], s["scale"], s["block"], width, score_cap=s["cap"], distance_slopes=s["slope"],
                                             window=s["window"])
    elif s["op"] == "prompt":
        paged_kernels.paged_scored_prefill_attention(*a, s["offsets"], s["tokens"], s["starts"], s["scale"], s["block"], width, score_cap=s["cap"],
                                                     distance_slopes=s["slope"], window=s["window"])
    else:
        paged_kernels.paged_shared_prefix_attention(*a, s["seq_lens"], s["group_offsets"], s["shared_lens"], s["scale"], s["block"], width)
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits, one row of the batch and one kv head after another
# ---------------------------------------------------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "norms":
        f64 = lambda t: None if t is None else t.double()  # noqa: E731
        x, r, w, pw, g = (f64(s[k]) for k in ("x", "residual", "weight", "post_weight", "gate"))
        if pw is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / c["hidden"] + 1e-6).sqrt() * (pw + c["offset"])
        r = r + c["scale"] * (x if g is None else x * g)
        return {"residual": r, "normed": r / (r.pow(2).sum(-1, keepdim=True) / c["hidden"] + 1e-6).sqrt() * (w + c["offset"])}
    group = c["hq"] // c["hkv"]
    out = torch.empty(s["query"].shape, dtype=torch.float64, device=s["query"].device)
    if c["op"] == "prompt":
        rows = list(zip(s["offsets"], s["tokens"], s["starts"]))
    else:
        rows = [(i, 1, n - 1) for i, n in enumerate(s["seq_lens"].tolist())]
    for i, (off, n, start) in enumerate(rows):
        pages = s["block_tables"][i, : -(-(start + n) // c["block"])].long()
        i_pos = torch.arange(start, start + n, device=out.device)[:, None]
        j_pos = torch.arange(start + n, device=out.device)[None, :]
        seen = j_pos <= i_pos
        if c.get("window"):
            seen &= j_pos > i_pos - c["window"]
        for h in range(c["hkv"]):
            k = s["k_cache"][pages, h].double().flatten(0, 1)[: start + n]
            v = s["v_cache"][pages, h].double().flatten(0, 1)[: start + n]
            for g in range(h * group, (h + 1) * group):
                x = s["query"][off:off + n, g].double() @ k.T * s["scale"]
                if c.get("cap"):
                    x = c["cap"] * torch.tanh(x / c["cap"])
                if s["slope"] is not None:
                    x = x - s["slope"][g].double() * (i_pos - j_pos)
                x = torch.softmax(x.masked_fill(~seen, -math.inf), dim=-1)
                out[off:off + n, g] = x @ v
    return out
