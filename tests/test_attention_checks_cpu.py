"""Host-side checks of the attention calls that need no GPU."""
import ctypes

import pytest
import torch

from reax_engine_b200 import _lib as L
from reax_engine_b200 import attention as A
from test_attention_cpu import BASE, call


def test_an_empty_output_shares_nothing():
    """Empty tensors all have the data pointer 0."""
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16)
    for out in (torch.empty(0, 4, 64, dtype=torch.bfloat16), q):
        assert A._output(out, q, (q, q, q)) is out
    t = torch.empty(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        A._output(t[1:], t[:2], (t,))


def test_rows_of_the_output_must_not_overlap():
    """Token and head strides that are each wide enough, together (100 tokens, 16 heads of 64)."""
    bad = [(64, 64), (128, 64), (512, 64), (1024 - 8, 64), (64, 128), (64, 6400 - 8), (128, 192), (64 * 7, 64 * 3)]
    good = [(1024, 64), (1032, 64), (2048, 128), (64, 6400), (72, 7200), (64, 1 << 20), (1 << 20, 64), (64 * 33, 64 * 2),
            (64 * 17, 64 * 2 * 17 + 64)]
    rows = lambda t, h: [i * t + j * h for i in range(100) for j in range(16)]  # noqa: E731
    for t, h in bad + good:
        at = sorted(rows(t, h))
        overlap = any(b - a < 64 for a, b in zip(at, at[1:]))
        assert call(out_stride=t, out_head_stride=h) == (L.ERR_MISALIGNED if overlap else L.ERR_WORKSPACE), (t, h)
    assert any(b - a < 64 for t, h in bad for a, b in zip(sorted(rows(t, h)), sorted(rows(t, h))[1:]))
    # inputs may (a broadcast or sliding view reads the same elements twice)
    assert call(k_stride=64) == L.ERR_WORKSPACE


def test_inputs_that_carry_derivatives():
    from torch.autograd import forward_ad
    x, y = torch.ones(2, 1, 64), torch.ones(2, 1, 64)
    A._no_gradients((x, y))
    with pytest.raises(ValueError):
        A._no_gradients((x, y.clone().requires_grad_()))
    with torch.no_grad():
        A._no_gradients((x, y.clone().requires_grad_()))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for ts in ((dual, y), (y, dual), (y, dual[:1])):
            with pytest.raises(ValueError):
                A._no_gradients(ts)
            with torch.no_grad(), pytest.raises(ValueError):
                A._no_gradients(ts)
        A._no_gradients((y, forward_ad.unpack_dual(dual).primal))
    A._no_gradients((x, y))


def test_half_a_prefix():
    import reax_engine_b200 as R
    t, c = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    for pk, pv in ((t, None), (None, t)):
        with pytest.raises(ValueError, match="go together"):
            R.shared_prefix_attention(t, t, t, pk, pv, c)


def test_a_scale_whose_product_with_log2_e_is_infinite():
    """2.4e38 log2(e) is past fp32's range: every weight would be NaN."""
    for s in (2.4e38, 2.9e38, 3.4e38):
        a = L.AttentionArgs(**{**BASE, "scale": s})
        assert L.lib().reaxmoe_attention_workspace_size(ctypes.byref(a)) == 0 and call(scale=s) == L.ERR_BAD_SHAPE
    assert call(scale=2.2e38) == L.ERR_WORKSPACE


def test_the_plan_that_other_tests_go_by():
    import random
    from attention_plan import plan
    rng = random.Random(3)
    for _ in range(3000):
        kv, d = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 256])
        hq = kv * rng.choice([1, 2, 4, 5, 8, 16, 17])
        seqs = rng.choice([1, 2, 7, 64, 300])
        nq = rng.choice([1, seqs, seqs + 1, seqs * 40])
        nk = rng.choice([nq, 16 * seqs - 1, 16 * seqs, 4095, 4096, 32767, 32768, 200000])
        prefix = rng.choice([0, 0, 1, 512, 513, 20000])
        a = L.AttentionArgs(**{**BASE, "q_tokens": nq, "k_tokens": nk, "seqs": seqs, "q_heads": hq, "kv_heads": kv, "head_dim": d,
                               "prefix": prefix})
        assert L.lib().reaxmoe_attention_workspace_size(ctypes.byref(a)) == plan(nq, nk, seqs, hq, kv, d, prefix).workspace
