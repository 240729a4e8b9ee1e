"""The norms and the vocabulary loss inside the LM, together as a training step uses them.

A two-layer model runs with the operators on the GPU; its twin has the CPU oracle as its cores
and the plain torch form of everything else, in float64.  fp32 end to end, with and without the
block options (norm after a block, gates, learned scale), checkpointed and not: loss within 1e-5
and every gradient within 1e-3 relative L2, the criteria of the model's other parity tests.
"""
from __future__ import annotations

import dataclasses

import pytest
import torch

from gpa_b200 import _lib
from gpa_b200.lm import GPALM, BlockOutput, GPALMConfig, RMSNorm
from gpa_b200.training_graph import GradientGraph
from lm_around import Adapted, Round, shard
from lm_oracle import oracle_lm
from parity_util import rel

pytestmark = pytest.mark.gpu

CFG = GPALMConfig(vocab_size=500, hidden_size=128, num_layers=2, num_heads=4, num_kv_heads=2,
                  head_dim=32, intermediate_size=256, slots=(16, 16, 32), chunk_size=64,
                  loss_chunk_size=48)
OPTIONS = [dict(post_norms=True), dict(block_gate="token"), dict(residual_scale=0.5),
           dict(post_norms=True, block_gate="channel", residual_scale=0.5)]


def _model(cfg, seed=0):
    torch.manual_seed(seed)
    m = GPALM(cfg)
    with torch.no_grad():
        for blk in m.blocks:
            blk.attn.conv.normal_(0., .3)
            for out in (blk.attn_out, blk.mlp_out):
                for p in out.parameters():
                    p.add_(torch.randn_like(p) * 0.1)
            for w in blk.attn.gpa.query_weight:
                w.normal_(0., .2)
    return m


@pytest.mark.parametrize("checkpointing", [False, True])
@pytest.mark.parametrize("options", OPTIONS)
def test_block_options_match_the_plain_form(options, checkpointing, cpu_threads):
    m = _model(dataclasses.replace(CFG, **options))
    twin = oracle_lm(m)
    ids = torch.randint(0, CFG.vocab_size, (2, 70), generator=torch.Generator().manual_seed(1))
    labels = ids.clone()
    labels[0, 3:9] = -100
    twin.train()
    ref, _ = twin(ids, labels=labels)
    ref.backward()
    gpu = m.cuda().train()
    gpu.gradient_checkpointing, gpu.autocast = checkpointing, False
    loss, _ = gpu(ids.cuda(), labels=labels.cuda())
    loss.backward()
    assert rel(loss, ref) <= 1e-5
    want = {n.replace("gpa.inner.", "gpa."): p.grad for n, p in twin.named_parameters() if p.grad is not None}
    got = {n: p.grad for n, p in gpu.named_parameters() if p.grad is not None}
    assert set(got) <= set(want)
    bad = {n: rel(g, want[n]) for n, g in got.items() if not rel(g, want[n]) <= 1e-3}
    assert not bad, bad


def test_state_dict_names_are_those_without_the_options():
    names = set(GPALM(CFG).state_dict())
    assert not any("attn_out" in n or "mlp_out" in n for n in names)
    assert {n.split("blocks.0.")[1] for n in set(_model(dataclasses.replace(CFG, **OPTIONS[3])).state_dict())
            - names if "blocks.0." in n} == {
        f"{b}_out.{p}" for b in ("attn", "mlp") for p in ("post.weight", "gate.weight", "gate.bias", "scale")}


@pytest.mark.parametrize("options", [{}, OPTIONS[3]])
def test_generation_paths_agree_and_use_the_kernels(options):
    m = _model(dataclasses.replace(CFG, **options), seed=2).cuda().eval()
    ids = torch.randint(0, CFG.vocab_size, (3, 70), generator=torch.Generator().manual_seed(3)).cuda()
    a = m.generate(ids, 6, fused_decode=True)
    _lib.profile_start()
    b = m.generate(ids, 6, fused_decode=False)
    counts = _lib.profile_stop()
    # Both paths compute in bf16 with kernels of their own, whose results are within 2e-2 relative
    # L2 of one another (the criterion of the bf16 parity tests).  A logit is n . w with |n| =
    # sqrt(hidden) after the final norm (weights 1), so two candidates may change places only if
    # their logits differ by at most 2e-2 |n| |w_a - w_b|; after that the sequences part.
    head = m.lm_head.weight.detach().float()
    for i in range(3):
        part = (a[i] != b[i]).nonzero()
        if len(part):
            k = int(part[0])
            with torch.no_grad():
                logits, _ = m(torch.cat((ids[i], a[i, :k]))[None])
            u, v = int(a[i, k]), int(b[i, k])
            margin = float((logits[0, -1, u] - logits[0, -1, v]).abs())
            assert margin <= 2e-2 * CFG.hidden_size ** .5 * float((head[u] - head[v]).norm()), (i, k, margin)
    # per call: the first norm, a q and a k norm a layer, a join after each of its two blocks
    assert counts["norm_fwd"][0] == 6 * (1 + 2 * (2 + 2))


def test_training_step_runs_the_kernels_under_autocast_and_in_a_graph():
    m = _model(CFG, seed=4).cuda().train()
    ids = torch.randint(0, CFG.vocab_size, (2, 64), generator=torch.Generator().manual_seed(5)).cuda()
    _lib.profile_start()
    loss, _ = m(ids, labels=ids)
    loss.backward()
    counts = _lib.profile_stop()
    assert {"norm_fwd", "norm_bwd", "loss_stats_tc5", "loss_probs_tc5", "loss_dx_tc5", "loss_dw_tc5"} <= set(counts)
    want = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}
    value = loss.detach().clone()
    del loss  # the eager graph is gone before the capture
    graph = GradientGraph(m, (torch.zeros(1, device="cuda"),), lambda _: (m(ids, labels=ids)[0], ids))
    got, _ = graph.replay(torch.zeros(1, device="cuda"))
    assert torch.equal(got, value)
    bad = {n: rel(p.grad, want[n]) for n, p in m.named_parameters()
           if p.grad is not None and not rel(p.grad, want[n]) <= 1e-2}
    assert not bad, bad


def test_no_label_at_all_gives_zero_loss_and_gradients():
    m = _model(CFG, seed=6).cuda().train()
    ids = torch.zeros(2, 5, dtype=torch.long, device="cuda")
    loss, _ = m(ids, labels=torch.full_like(ids, -100))
    loss.backward()
    assert float(loss) == 0 and not m.embed.weight.grad.any()


def _step(m, ids, labels):
    m.zero_grad(set_to_none=True)
    loss, _ = m(ids, labels=labels)
    loss.backward()
    return loss.detach(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("checkpointing", [False, True])
@pytest.mark.parametrize("options", [{}, OPTIONS[3]])
@pytest.mark.parametrize("what", ["blocks", "norms", "head", "posts"])
def test_hooked_modules_are_called(what, options, checkpointing):
    # a head of its own: the embedding reads its table outside the head's forward
    m = _model(dataclasses.replace(CFG, tie_embeddings=False, **options), seed=7).cuda().train()
    m.gradient_checkpointing, m.autocast = checkpointing, False
    ids = torch.randint(0, CFG.vocab_size, (2, 70), generator=torch.Generator().manual_seed(8)).cuda()
    want, grads = _step(m, ids, ids)
    some = {"blocks": list(m.blocks), "head": [m.lm_head],
            "norms": [n for b in m.blocks for n in (b.input_norm, b.post_norm)] + [m.norm],
            "posts": [o.post for b in m.blocks for o in (b.attn_out, b.mlp_out) if o.post is not None]}[what]
    calls, handles = [], [mod.register_forward_hook(lambda mod, a, o: calls.append(mod)) for mod in some]
    got, again = _step(m, ids, ids)
    assert {id(c) for c in calls} == {id(mod) for mod in some}
    assert rel(got, want) <= 1e-5
    bad = {n: rel(again[n], g) for n, g in grads.items() if not rel(again[n], g) <= 1e-3}
    assert not bad and set(again) == set(grads), bad
    for h in handles:
        h.remove()
    back = [shard(mod) for mod in some]
    with torch.no_grad():
        assert rel(m(ids, labels=ids)[0], want) <= 1e-5
    for f in back:
        f()


@pytest.mark.parametrize("head", ["adapted", "biased", "wrapped"])
def test_replaced_heads_are_called(head, cpu_threads):
    m = _model(CFG, seed=9)
    m.lm_head.weight = torch.nn.Parameter(m.lm_head.weight.detach().clone())
    if head == "adapted":
        m.lm_head = Adapted(m.lm_head)
    elif head == "biased":
        m.lm_head.bias = torch.nn.Parameter(torch.randn(CFG.vocab_size, generator=torch.Generator().manual_seed(1)))
    else:
        m.lm_head = Round(m.lm_head)
    twin = oracle_lm(m).train()
    ids = torch.randint(0, CFG.vocab_size, (2, 70), generator=torch.Generator().manual_seed(10))
    ref, wanted = _step(twin, ids, ids)
    gpu = m.cuda().train()
    gpu.autocast = False
    loss, got = _step(gpu, ids.cuda(), ids.cuda())
    assert rel(loss, ref) <= 1e-5
    bad = {n: rel(g, wanted[n.replace("gpa.", "gpa.inner.")]) for n, g in got.items()
           if not rel(g, wanted[n.replace("gpa.", "gpa.inner.")]) <= 1e-3}
    assert not bad, bad


def test_every_option_gets_its_gradient():
    m = _model(dataclasses.replace(CFG, **OPTIONS[3]), seed=11).cuda().train()
    ids = torch.randint(0, CFG.vocab_size, (2, 70), generator=torch.Generator().manual_seed(12)).cuda()
    grads = _step(m, ids, ids)[1]
    wanted = {n for n, _ in m.named_parameters() if "attn_out" in n or "mlp_out" in n or "norm" in n}
    assert wanted and wanted <= set(grads) and all(grads[n].any() for n in wanted)


def _expected(x, head, labels):
    z = x.double().flatten(0, 1) @ head.double().T
    y = torch.nn.functional.pad(labels[:, 1:], (0, 1), value=-100).flatten()
    return torch.nn.functional.cross_entropy(z, y, ignore_index=-100)


@pytest.mark.parametrize("tokens,grad", [((1 << 22) + 2, True), (9, False), (9, True)])
def test_losses_of_every_size_are_answered(tokens, grad):
    """More tokens than linear_cross_entropy takes in a call, and few: 1e-5 relative, fp32's
    rounding over 8 channels and a mean with room."""
    cfg = dataclasses.replace(CFG, vocab_size=16, hidden_size=8, num_layers=0, loss_chunk_size=1 << 20)
    m = GPALM(cfg).cuda().eval()
    g = torch.Generator().manual_seed(13)
    x = torch.randn(1, tokens, 8, generator=g).cuda().requires_grad_(grad)
    labels = torch.randint(0, 16, (1, tokens), generator=g).cuda()
    with torch.set_grad_enabled(grad):
        loss = m._loss(x, labels)
    ref = _expected(x.detach(), m.lm_head.weight.detach(), labels)
    assert loss.dtype == torch.float32 and rel(loss, ref) <= 1e-5
    if grad:
        (dx,) = torch.autograd.grad(loss, x)
        assert dx.isfinite().all() and dx[:, :-1].any(-1).all() and not dx[:, -1].any()


def test_one_token_with_its_label_has_no_loss():
    m = _model(CFG, seed=14).cuda().train()
    ids = torch.zeros(3, 1, dtype=torch.long, device="cuda")
    _lib.profile_start()
    loss, grads = _step(m, ids, ids)
    counts = _lib.profile_stop()
    assert float(loss) == 0 and not any("loss" in k for k in counts)
    assert loss.dtype == torch.float32 and not any(g.any() for g in grads.values())


def test_a_model_without_layers_generates():
    m = GPALM(dataclasses.replace(CFG, num_layers=0)).cuda().eval()
    ids = torch.randint(0, CFG.vocab_size, (2, 5), generator=torch.Generator().manual_seed(15)).cuda()
    assert torch.equal(m.generate(ids, 3), m.generate(ids, 3, fused_decode=False))


def test_the_model_s_norm_keeps_forward_mode_and_transforms():
    norm = RMSNorm(48, 1e-6).cuda()
    g = torch.Generator().manual_seed(16)
    x, t = (torch.randn(5, 48, generator=g).cuda() for _ in range(2))
    out, tangent = torch.func.jvp(norm, (x,), (t,))
    xd, td = x.double(), t.double()
    r = 1 / (xd.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    want = td * r - xd * r ** 3 * (xd * td).mean(-1, keepdim=True)
    # each term carries a few fp32 roundings and a mean of 48: 64 of them are room enough
    mag = (td.abs() * r + xd.abs() * r ** 3 * (xd * td).abs().mean(-1, keepdim=True))
    assert ((tangent.double() - want).abs() <= 64 * 2.0 ** -24 * mag).all()
    assert torch.allclose(torch.func.vmap(norm)(x), norm(x), atol=0, rtol=1e-5)


@pytest.mark.parametrize("stream,update", [(torch.float16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16)])
def test_stream_has_the_type_of_the_addition(stream, update):
    """As of x + y: half-precision weights under bf16 autocast leave an fp32 stream."""
    out, norm = BlockOutput(CFG).cuda(), RMSNorm(128, 1e-6).cuda()
    g = torch.Generator().manual_seed(17)
    x, y = torch.randn(5, 128, generator=g).cuda().to(stream), torch.randn(5, 128, generator=g).cuda().to(update)
    s, n = out.add_and_norm(x, y, None, norm, torch.bfloat16)
    assert s.dtype == (x + y).dtype and torch.equal(s, x + y) and n.dtype == torch.bfloat16
