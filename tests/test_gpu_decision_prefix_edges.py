"""DecisionModel's prefixes at their edges: prompts that add nothing to the prefix."""
import pytest
import torch

from test_gpu_decision import small_cfg

pytestmark = pytest.mark.gpu


def prefixed(seed=3, length=23, lens=(4, 9, 2)):
    from reax_engine_b200.decision import DecisionModel, synthetic_prompts
    cfg = small_cfg(layers=2)
    model = DecisionModel(cfg, "cuda", seed=seed, attention="native")
    head, cu = synthetic_prompts(1, length, length, cfg.vocab, seed=seed)
    model.calibrate(head.cuda(), cu.cuda())
    tails = [synthetic_prompts(1, n, n, cfg.vocab, seed=seed + n)[0] for n in lens]
    return model, head, tails, model.prefill_prefix(head.cuda()), torch.tensor([5, 17, 100, 400]).cuda()


def packed(parts):
    cu = torch.tensor([0] + [p.numel() for p in parts]).cumsum(0).to(torch.int32).cuda()
    return torch.cat(parts).cuda() if parts else torch.zeros(0, dtype=torch.long), cu


@pytest.mark.parametrize("where", [(0,), (1,), (3,), (0, 1, 3, 5), (2, 2)])
def test_prompts_that_add_nothing(where):
    """A prompt of no tokens has the answer of the prefix as a prompt, and the others have theirs. The products with the option
    embeddings are of other shapes, so that the logits (below 4, bf16) may differ by a step, 2^-6: 2^-5 relative in a weight."""
    model, head, tails, state, opts = prefixed()
    none = torch.zeros(0, dtype=torch.long)
    parts = list(tails)
    for w in where:
        parts.insert(w, none)
    got = model.forward(*packed(parts), opts, prefix=state)
    alone = model.forward(head.cuda(), packed([head])[1], opts)
    others = iter(model.forward(*packed(tails), opts, prefix=state))
    assert got.shape == (len(parts), 4)
    for p, row in zip(parts, got):
        want = alone[0] if p.numel() == 0 else next(others)
        assert (row - want).abs().max() <= 2.0 ** -5 * want.max()
    # distinct answers, so that one taken from another prompt would show
    assert (alone[0] - model.forward(*packed(tails), opts, prefix=state)).abs().amax(-1).min() > 2.0 ** -4


@pytest.mark.parametrize("n", [1, 3])
def test_only_prompts_that_add_nothing(n):
    model, head, _, state, opts = prefixed()
    got = model.forward(torch.zeros(0, dtype=torch.long), torch.zeros(n + 1, dtype=torch.int32), opts, prefix=state)
    alone = model.forward(head.cuda(), packed([head])[1], opts)
    assert got.shape == (n, 4) and (got - alone).abs().max() <= 2.0 ** -5


def test_a_prefix_without_its_last_row_is_refused_for_such_prompts():
    from reax_engine_b200.decision import PrefixState
    model, _, tails, state, opts = prefixed()
    bare = PrefixState(state.length, state.keys, state.values)
    with pytest.raises(ValueError):
        model.forward(*packed([tails[0], torch.zeros(0, dtype=torch.long)]), opts, prefix=bare)
    model.forward(*packed(tails), opts, prefix=bare)


def test_a_wait_that_ran_out_is_not_passed_over(monkeypatch):
    """Every attention call is given the model's status word; a code in it makes the results NaN and the next call raise, keeps a
    prefix from being handed out, and is gone then. (The code is written by the host here.)"""
    from reax_engine_b200 import _lib as L
    from reax_engine_b200 import decision
    model, head, tails, state, opts = prefixed()
    ids, cu = packed(tails)
    good, good_prefix = model.forward(ids, cu, opts), model.forward(ids, cu, opts, prefix=state)
    calls = []
    for name in ("prompt_attention", "shared_prefix_attention"):
        def failing(*a, real=getattr(decision, name), status, **kw):
            calls.append(status)
            if len(calls) % 2:                                 # of the two layers the first
                status.fill_(L.ERR_DEVICE_TIMEOUT)
            return real(*a, status=status, **kw)
        monkeypatch.setattr(decision, name, failing)
    for prefix in (None, state):
        assert torch.isnan(model.forward(ids, cu, opts, prefix=prefix)).all()
        with pytest.raises(L.ReaxMoEError) as e:
            model.forward(ids, cu, opts)
        assert e.value.code == L.ERR_DEVICE_TIMEOUT and len(calls) % 2 == 0
    with pytest.raises(L.ReaxMoEError):
        model.prefill_prefix(head.cuda())
    assert torch.isnan(model.forward(ids, cu, opts)).all() and model.read_status() == L.ERR_DEVICE_TIMEOUT
    before = list(model.input_amax)
    with pytest.raises(L.ReaxMoEError):
        model.calibrate(ids, cu)
    assert model.input_amax == before
    monkeypatch.undo()
    assert model.read_status() == 0
    assert torch.equal(model.forward(ids, cu, opts), good)
    assert torch.equal(model.forward(ids, cu, opts, prefix=state), good_prefix)


def test_lengths_that_do_not_fit_the_tokens_are_refused():
    """Tokens behind the last prompt, prompts behind the last token, a start that is not 0, and lengths that fall: positions and
    rows would be taken from outside the batch."""
    model, _, tails, state, opts = prefixed()
    ids, cu = packed(tails)
    bad = [(torch.cat([ids, ids[:3]]), cu), (ids[:-1], cu), (ids, cu + 1), (ids, cu[[0, 2, 1, 3]]), (ids[:4], cu[:1].repeat(3))]
    for t, c in bad:
        for prefix in (None, state):
            with pytest.raises(ValueError):
                model.forward(t, c, opts, prefix=prefix)
    model.forward(ids, cu, opts, prefix=state)
