"""What reaxmoe_attention and its Python calls refuse before any kernel runs (no GPU)."""
import ctypes

import pytest
import torch

import reax_engine_b200 as R
from reax_engine_b200 import _lib as L

BASE = dict(q=16, k=16, v=16, prefix_k=16, prefix_v=16, cu_q=16, cu_k=16, out=16, q_stride=1024, q_head_stride=64, k_stride=512,
            k_head_stride=64, v_stride=512, v_head_stride=64, prefix_k_stride=512, prefix_k_head_stride=64, prefix_v_stride=512,
            prefix_v_head_stride=64, out_stride=1024, out_head_stride=64, q_tokens=100, k_tokens=100, prefix=10, seqs=2,
            q_heads=16, kv_heads=8, head_dim=64, dtype=L.BF16, causal=1, window=0, scale=0.125)


def call(**kw):
    """With no workspace: sizes, pointers and strides are checked before it, so a good call ends there."""
    a = L.AttentionArgs(**{**BASE, **kw})
    return L.lib().reaxmoe_attention(ctypes.byref(a), None, 0, None)


def test_a_good_call_needs_its_workspace():
    assert call() == L.ERR_WORKSPACE
    a = L.AttentionArgs(**BASE)
    assert L.lib().reaxmoe_attention_workspace_size(ctypes.byref(a)) >= 16
    assert L.lib().reaxmoe_attention(None, None, 0, None) == L.ERR_NULL
    assert L.lib().reaxmoe_attention_workspace_size(None) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=96), L.ERR_BAD_SHAPE), (dict(q_heads=12, kv_heads=8), L.ERR_BAD_SHAPE), (dict(kv_heads=0), L.ERR_BAD_SHAPE),
    (dict(q_heads=129, kv_heads=1), L.ERR_BAD_SHAPE),
    (dict(seqs=-1), L.ERR_BAD_SHAPE), (dict(q_tokens=-1), L.ERR_BAD_SHAPE), (dict(k_tokens=1 << 31), L.ERR_BAD_SHAPE),
    (dict(k_tokens=1 << 30, prefix=1 << 30), L.ERR_BAD_SHAPE), (dict(q_tokens=(1 << 31) - 70000), L.ERR_BAD_SHAPE),
    (dict(prefix=-5), L.ERR_BAD_SHAPE), (dict(dtype=2), L.ERR_UNSUPPORTED), (dict(causal=2), L.ERR_BAD_SHAPE),
    (dict(window=-1), L.ERR_BAD_SHAPE), (dict(window=5, causal=0), L.ERR_BAD_SHAPE), (dict(scale=0.0), L.ERR_BAD_SHAPE),
    (dict(scale=-1.0), L.ERR_BAD_SHAPE), (dict(scale=float("nan")), L.ERR_BAD_SHAPE), (dict(scale=float("inf")), L.ERR_BAD_SHAPE)])
def test_bad_sizes(kw, code):
    a = L.AttentionArgs(**{**BASE, **kw})
    assert L.lib().reaxmoe_attention_workspace_size(ctypes.byref(a)) == 0
    assert call(**kw) == code and L.last_error()


@pytest.mark.parametrize("name", ["q", "k", "v", "prefix_k", "prefix_v", "cu_q", "cu_k", "out"])
def test_missing_and_misaligned_tensors(name):
    assert call(**{name: None}) == L.ERR_NULL
    if not name.startswith("cu"):
        assert call(**{name: 24}) == L.ERR_MISALIGNED


@pytest.mark.parametrize("name", ["q", "k", "v", "prefix_k", "prefix_v", "out"])
def test_bad_strides(name):
    assert call(**{name + "_stride": 516}) == L.ERR_MISALIGNED
    assert call(**{name + "_head_stride": 68}) == L.ERR_MISALIGNED
    assert call(**{name + "_head_stride": 32}) == L.ERR_MISALIGNED        # heads that overlap
    assert call(**{name + "_stride": 0}) == L.ERR_MISALIGNED              # tokens that overlap
    assert call(**{name + "_stride": -1024}) == L.ERR_MISALIGNED
    assert call(**{name + "_stride": 1 << 38}) == L.ERR_MISALIGNED        # past a tensor map's range


def test_nothing_to_do():
    assert call(q_tokens=0, q=None, out=None) == L.OK
    assert call(seqs=0) == L.OK
    # tensors that are not read may be missing
    assert call(prefix=0, prefix_k=None, prefix_v=None) == L.ERR_WORKSPACE
    assert call(k_tokens=0, k=None, v=None) == L.ERR_WORKSPACE


def test_python_calls_take_cuda_tensors_only():
    t = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    c = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError):
        R.prompt_attention(t, t, t, c)
    with pytest.raises(ValueError):
        R.shared_prefix_attention(t, t, t, t, t, c)
