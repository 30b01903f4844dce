"""GPU: the decoder stack with capped scores, windows, distance biases, norms behind its blocks and shared prefixes — the
operators together, as a step uses them — against a plain restatement in 64 bits."""
import pytest
import torch
import torch.nn.functional as F

from nanopd_b200 import decoder_step, paged_forward, paged_kernels
from oracle import paged_oracle, shaped_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BASE = dict(num_layers=3, hidden=256, ffn=512, vocab=1000, num_q_heads=4, num_kv_heads=2, head_dim=64, rope_theta=1e4)
SHAPES = {
    "capped": decoder_step.DecoderShape(**BASE, score_cap=5.0, window=24, window_every=2, post_norms=True, norm_offset=1.0),
    "biased": decoder_step.DecoderShape(**BASE, distance_bias=True, residual_scale=0.4),
    "window": decoder_step.DecoderShape(**BASE, window=17, post_norms=True, residual_scale=0.7),
}


def make_batch(dtype, ctx, shape, steps_ahead=4, seed=0):
    torch.manual_seed(seed)
    B = 16
    ctx = torch.tensor(ctx, dtype=torch.int32)
    nblk = [(int(c) + steps_ahead + B) // B for c in ctx]
    pool = sum(nblk) + 2
    perm = torch.randperm(pool)
    tables = torch.zeros(len(ctx), max(nblk), dtype=torch.int32)
    o = 0
    for i, n in enumerate(nblk):
        tables[i, :n] = perm[o:o + n].to(torch.int32)
        o += n
    kc, vc = (torch.randn(shape.num_layers, pool, shape.num_kv_heads, B, shape.head_dim).to(dtype) for _ in range(2))
    return kc, vc, tables, ctx, torch.randint(0, shape.vocab, (len(ctx),))


def plain_step(model, kc, vc, tables, ctx, tokens):
    """One decode step on the CPU: 64-bit products on the 16-bit weights, rounded where the step rounds."""
    s, dt = model.shape, model.dtype
    cpu = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    mm = lambda a, w: (a.double() @ cpu(w).double().T).to(dt)  # noqa: E731
    x = cpu(model.embed)[tokens]
    pos = ctx.long()
    cos, sin = cpu(model.cos_table)[pos], cpu(model.sin_table)[pos]
    hq_d, hkv_d, S = s.num_q_heads * s.head_dim, s.num_kv_heads * s.head_dim, tokens.numel()
    first = cpu(model.layers[0]["in_norm"])
    h = shaped_oracle.residual_norms(torch.zeros_like(x), x, first, eps=s.eps, weight_offset=s.norm_offset)[1].to(dt)
    for li, L in enumerate(model.layers):
        qkv = mm(h, L["w_qkv"])
        q, k, v = (t.reshape(S, -1, s.head_dim) for t in qkv.split([hq_d, hkv_d, hkv_d], dim=1))
        q_rot = paged_oracle.qk_norm_rope_store(q, k, v, cos, sin, kc[li], vc[li], tables, ctx, cpu(L["q_norm"]), cpu(L["k_norm"]), s.eps)
        window = s.window if s.window and li % s.window_every == 0 else 0
        attn, _, _ = shaped_oracle.attend_single(q_rot, kc[li], vc[li], tables, ctx + 1, model.scale, s.score_cap, cpu(model.slopes), window)
        y = mm(attn.to(dt).reshape(S, hq_d), L["w_o"])
        r, h, _ = shaped_oracle.residual_norms(y, x, cpu(L["post_norm"]), cpu(L["attn_out_norm"]), None, s.residual_scale, s.eps, s.norm_offset)
        x, h = r.to(dt), h.to(dt)
        gu = mm(h, L["w_gate_up"])
        y = mm(F.silu(gu[:, :s.ffn]) * gu[:, s.ffn:], L["w_down"])
        following = model.layers[li + 1]["in_norm"] if li + 1 < len(model.layers) else model.final_norm
        r, h, _ = shaped_oracle.residual_norms(y, x, cpu(following), cpu(L["mlp_out_norm"]), None, s.residual_scale, s.eps, s.norm_offset)
        x, h = r.to(dt), h.to(dt)
    return h.double() @ cpu(model.lm_head).double().T


@pytest.mark.parametrize("name", sorted(SHAPES))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_step_matches_a_plain_restatement(kernels, dtype, name):
    model = decoder_step.SyntheticDecoder(DEV, SHAPES[name], dtype, seed=1, max_position=512)
    kc, vc, tables, ctx, tokens = make_batch(dtype, [5, 31, 16, 270, 64], SHAPES[name])
    model.attach_batch(kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx.to(DEV), tokens.to(DEV))
    model.step()
    torch.cuda.synchronize()
    want = plain_step(model, kc, vc, tables, ctx, tokens)
    got = model.logits.double().cpu()
    # three layers of 16-bit activations: each of the ~12 roundings on a row's way is half a step of the type
    off = (got - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(off.max()) < 24 * torch.finfo(dtype).eps / 2, off
    assert model.launches_per_step() == 4 * 3 + 1


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_graph_replays_equal_eager_steps(kernels, name):
    dtype = torch.bfloat16
    model = decoder_step.SyntheticDecoder(DEV, SHAPES[name], dtype, seed=2, max_position=512)
    kc, vc, tables, ctx, tokens = make_batch(dtype, [5, 31, 16, 270], SHAPES[name], seed=3)
    model.attach_batch(kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx.to(DEV), tokens.to(DEV))
    eager = []
    for _ in range(3):
        model.step()
        eager.append((model.token_ids.clone(), model.logits.clone()))
    model.attach_batch(kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx.to(DEV), tokens.to(DEV))
    model.capture()
    for t, l in eager:
        model.replay()
        torch.cuda.synchronize()
        assert torch.equal(model.token_ids, t) and torch.equal(model.logits, l)


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_a_prompt_in_chunks_beside_a_decode_batch(kernels, name):
    """A prompt of 70 tokens in one chunk, in two, and fed token by token ends in the same logits up to the type's rounding."""
    dtype, shape = torch.float16, SHAPES[name]
    model = decoder_step.SyntheticDecoder(DEV, shape, dtype, seed=4, max_position=512)
    kc, vc, tables, ctx, tokens = make_batch(dtype, [5, 90], shape, seed=5)
    pool = kc.size(1)
    grow = lambda c: torch.cat((c, torch.zeros(c.size(0), 6, *c.shape[2:], dtype=dtype)), dim=1).to(DEV)  # noqa: E731
    table, prompt = list(range(pool, pool + 6)), torch.randint(0, shape.vocab, (70,))
    decodes = [{"block_table": tables[i, :(int(ctx[i]) + 16) // 16].tolist(), "position": int(ctx[i])} for i in range(2)]
    chunk = lambda start, n, dec: {"num_prefill_tokens": n, "num_decode_tokens": len(dec), "decodes": dec,  # noqa: E731
                                   "prefills": [{"block_table": table, "start_position": start, "num_tokens": n}]}
    k1, v1 = grow(kc), grow(vc)
    whole = model.mixed_step(chunk(0, 70, decodes), torch.cat((prompt, tokens)).to(DEV), k1, v1, overlap=False)
    k2, v2 = grow(kc), grow(vc)
    model.mixed_step(chunk(0, 40, []), prompt[:40].to(DEV), k2, v2)
    halves = model.mixed_step(chunk(40, 30, []), prompt[40:].to(DEV), k2, v2)
    k3, v3 = grow(kc), grow(vc)
    for i in range(70):
        step = {"num_prefill_tokens": 0, "num_decode_tokens": 1, "prefills": [], "decodes": [{"block_table": table, "position": i}]}
        single = model.mixed_step(step, prompt[i:i + 1].to(DEV), k3, v3)
    torch.cuda.synchronize()
    for other in (halves[0], single[0]):
        # both sides are as far from the exact logits as the step above may be
        assert float((other.float() - whole[0].float()).norm() / whole[0].float().norm()) < 2 * 24 * torch.finfo(dtype).eps / 2
    dec = {"num_prefill_tokens": 0, "num_decode_tokens": 2, "prefills": [], "decodes": decodes}
    alone = model.mixed_step(dec, tokens.to(DEV), grow(kc), grow(vc))
    assert float((alone.float() - whole[1:].float()).norm() / alone.float().norm()) < 2 * 24 * torch.finfo(dtype).eps / 2


def test_shaped_attention_steps_reach_the_shaped_operators(kernels):
    """``paged_attention_step`` with the shaping's arguments, against the operators called one by one."""
    torch.manual_seed(0)
    hq, hkv, d, B = 8, 2, 128, 16
    kc, vc = (torch.randn(40, hkv, B, d, device=DEV).to(torch.float16) for _ in range(2))
    ctx = {"num_prefill_tokens": 50, "num_decode_tokens": 2,
           "prefills": [{"block_table": list(range(5)), "start_position": 20, "num_tokens": 50}],
           "decodes": [{"block_table": list(range(10, 20)), "position": 140}, {"block_table": list(range(20, 23)), "position": 33}]}
    q, k, v = (torch.randn(1, h, 52, d, device=DEV).to(torch.float16) for h in (hq, hkv, hkv))
    shape = dict(score_cap=6.0, distance_slopes=torch.rand(hq, device=DEV), window=30)
    sc = paged_forward.build_step_context(ctx, DEV)
    out = paged_forward.paged_attention_step(sc, q, k, v, kc, vc, 0.1, overlap=False, **shape)[0].view(52, hq, d)
    tokens_major = q[0].transpose(0, 1).contiguous()
    want = torch.empty_like(tokens_major)
    paged_kernels.paged_scored_prefill_attention(want[:50], tokens_major[:50], kc, vc, sc.prefill_tables, [0], [50], [20], 0.1, B, 5, **shape)
    paged_kernels.paged_scored_attention(want[50:], tokens_major[50:], kc, vc, sc.decode_tables, sc.decode_seq_lens, 0.1, B,
                                         sc.decode_tables.size(1), **shape)
    assert torch.equal(out, want)


def test_shared_prefixes_in_a_captured_decoder(kernels):
    """A batch of 40 sequences behind 512 shared tokens, with and without being told so: the same logits up to rounding, in a
    captured step too; a batch that is told about groups it may not have is refused."""
    dtype = torch.float16
    shape = decoder_step.DecoderShape(**{**BASE, "num_q_heads": 16, "num_kv_heads": 8})
    model = decoder_step.SyntheticDecoder(DEV, shape, dtype, seed=7, max_position=1024)
    S, B, shared = 40, 16, 512
    ctx = torch.tensor([shared + 3 + 5 * i for i in range(S)], dtype=torch.int32)
    total = shared // B
    rows = []
    for c in ctx.tolist():
        own = (c + 4) // B + 1 - shared // B
        rows.append(list(range(shared // B)) + list(range(total, total + own)))
        total += own
    tables = torch.zeros(S, 160, dtype=torch.int32)              # a wide table: the batch is no small one by its bound
    for i, r in enumerate(rows):
        tables[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
    kc, vc = (torch.randn(shape.num_layers, total, shape.num_kv_heads, B, shape.head_dim, device=DEV).to(dtype) for _ in range(2))
    tokens = torch.randint(0, shape.vocab, (S,), device=DEV)
    groups = dict(group_offsets=torch.tensor([0, S], dtype=torch.int32, device=DEV), shared_lens=torch.tensor([shared], dtype=torch.int32, device=DEV))
    runs = []
    for kw, captured in (({}, False), (groups, False), (groups, True)):
        model.attach_batch(kc.clone(), vc.clone(), tables.to(DEV), ctx.to(DEV), tokens, **kw)
        if captured:
            model.capture()
        model.replay() if captured else model.step()
        torch.cuda.synchronize()
        runs.append(model.logits.clone())
    assert torch.equal(runs[1], runs[2])
    off = (runs[1].float() - runs[0].float()).norm(dim=-1) / runs[0].float().norm(dim=-1)
    assert float(off.max()) < 2 * 24 * torch.finfo(dtype).eps / 2
    with pytest.raises(RuntimeError, match="belong together"):
        model.attach_batch(kc, vc, tables.to(DEV), ctx.to(DEV), tokens, shared_lens=groups["shared_lens"])
