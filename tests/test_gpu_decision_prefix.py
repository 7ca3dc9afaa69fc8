"""The decision forward on this library's own attention, and on prompts that continue a shared prefix, against the CPU oracle:
every attention block from the GPU's own input to it (rel-L2 5e-3, the bar of the flash-attention model: bf16 weights in P V
against an fp32 softmax). Chained, such models drift apart at the level of bf16 roundings (routing swaps, NVFP4 codes that
flip), so whole forwards are held to the bar of the independent chain, 0.2 in probability."""
import pytest
import torch

from oracle import decision_oracle as D
from test_gpu_decision import cfg3_shapes, export, rel_l2, small_cfg

pytestmark = pytest.mark.gpu


def logs(model, f):
    model.layer_log = []
    out = f()
    got = [{k: v.cpu() for k, v in e.items()} if isinstance(e, dict) else e.cpu() for e in model.layer_log]
    model.layer_log = None
    return out, got


@pytest.mark.parametrize("shapes,n_prompts,lens,seed", [("small", 6, (10, 60), 1), ("cfg3", 3, (64, 300), 3)])
def test_native_attention_blocks_match_the_oracle(shapes, n_prompts, lens, seed):
    from reax_engine_b200.decision import DecisionModel, synthetic_prompts
    cfg = small_cfg(layers=3) if shapes == "small" else cfg3_shapes()
    model = DecisionModel(cfg, "cuda", seed=seed, attention="native")
    ids, cu = synthetic_prompts(n_prompts, *lens, cfg.vocab, seed=seed)
    model.calibrate(ids.cuda(), cu.cuda())
    opts = torch.tensor([5, 17, 100, 400]).cuda()
    p, got = logs(model, lambda: model.forward(ids.cuda(), cu.cuda(), opts))
    assert torch.allclose(p.sum(-1), torch.ones(n_prompts, dtype=torch.float64, device="cuda"))
    W, last = export(model), cu.long()[1:] - 1
    for i in range(cfg.layers):
        r = D.attention_block(W, cfg, i, got[i]["x"], cu)
        assert rel_l2(got[i]["r"], r[last] if i == cfg.layers - 1 else r) <= 5e-3, f"layer {i}"


@pytest.mark.parametrize("shapes,length,lens,seed", [("small", 37, (1, 30), 2), ("small", 3, (5, 20), 4), ("cfg3", 200, (3, 150), 5)])
def test_prompts_that_continue_a_prefix(shapes, length, lens, seed, capsys):
    from reax_engine_b200.decision import DecisionModel, synthetic_prompts
    cfg = small_cfg(layers=2) if shapes == "small" else cfg3_shapes(router_std=0.5)
    model = DecisionModel(cfg, "cuda", seed=seed, attention="native")
    ids, cu = synthetic_prompts(4, *lens, cfg.vocab, seed=seed)
    head, _ = synthetic_prompts(1, length, length, cfg.vocab, seed=seed + 100)
    parts = [torch.cat([head, ids[a:b]]) for a, b in zip(cu[:-1], cu[1:])]
    whole = torch.cat(parts)
    cu_whole = torch.tensor([0] + [len(t) for t in parts]).cumsum(0).to(torch.int32)
    model.calibrate(whole.cuda(), cu_whole.cuda())
    opts = torch.tensor([5, 17, 100, 400]).cuda()
    p_whole = model.forward(whole.cuda(), cu_whole.cuda(), opts)
    state, before = logs(model, lambda: model.prefill_prefix(head.cuda()))
    assert state.length == length and len(state.keys) == len(state.values) == cfg.layers
    p, after = logs(model, lambda: model.forward(ids.cuda(), cu.cuda(), opts, prefix=state))
    assert torch.equal(p, model.forward(ids.cuda(), cu.cuda(), opts, prefix=state))          # the state is not used up
    W = export(model)
    for i in range(cfg.layers):
        x = torch.cat([torch.cat([before[i]["x"], after[i]["x"][a:b]]) for a, b in zip(cu[:-1], cu[1:])])
        r = D.attention_block(W, cfg, i, x, cu_whole)
        mine = torch.cat([r[b - (cu[j + 1] - cu[j]):b] for j, b in enumerate(cu_whole[1:])])
        if i == cfg.layers - 1:
            mine = mine[cu.long()[1:] - 1]
        assert rel_l2(after[i]["r"], mine) <= 5e-3, f"layer {i}"
        if i < cfg.layers - 1:
            assert rel_l2(before[i]["r"], r[:length]) <= 5e-3, f"layer {i}, prefix"
    err = (p - p_whole).abs().max().item()
    with capsys.disabled():
        print(f"\n[decision prefix] after the prefix against the whole prompts: max |dp| = {err:.2e}")
    assert err < 0.2


def test_refusals():
    from reax_engine_b200.decision import DecisionModel, PrefixState, synthetic_prompts
    cfg = small_cfg()
    with pytest.raises(ValueError):
        DecisionModel(cfg, "cuda", attention="other")
    model = DecisionModel(cfg, "cuda", attention="native")
    with pytest.raises(ValueError):
        model.prefill_prefix(torch.zeros(0, dtype=torch.long))
    ids, cu = synthetic_prompts(2, 5, 9, cfg.vocab)
    with pytest.raises(ValueError):
        model.forward(ids, cu, torch.tensor([1, 2]), prefix=PrefixState(4, [], []))
