"""Generation steps on each of their paths, which the sizes of a call decide (attention_plan): own keys alone or behind a prefix
in one or several parts, joined by a warp or by a block a row; one and several rows a sequence; sequences of more rows than a
unit takes; non-finite values that rows do not see. Tolerances: those of test_gpu_attention."""
import pytest
import torch

from attention_plan import plan
from test_gpu_attention import check, cu, dev, reference, tensors

pytestmark = pytest.mark.gpu

SEVERAL = ((2, 0, 1, 0, 2), (700, 30, 900, 1, 1200))             # rows of a sequence; others without any
LONG = ((1, 1), (3000, 2500))                                   # many units a row
SHORT = ((1,) * 100, tuple(30 + 17 * i % 50 for i in range(100)))
MANY = ((20, 1) + (0,) * 23, (1500, 3000) + (3,) * 23)          # 20 rows x group: more than a unit takes


def run(q_lens, k_lens, hq, hk, d, dtype, prefix, window, parts, join_warps, seed, causal=True):
    import reax_engine_b200 as R
    cq, ck = cu(q_lens), cu(k_lens)
    p = plan(cq[-1], ck[-1], len(q_lens), hq, hk, d, prefix)
    assert p.few and join_warps in (None, p.join_warps) and (not prefix or p.parts == parts), p
    q, k, v, pk, pv = tensors(cq[-1], ck[-1], hq, hk, d, dtype, seed, prefix)
    kw = dict(window=window, causal=causal, return_lse=True)
    o, lse = (R.shared_prefix_attention(q, k, v, pk, pv, dev(cq), dev(ck), **kw) if prefix
              else R.prompt_attention(q, k, v, dev(cq), dev(ck), **kw))
    check(o, reference(q, k, v, cq, ck, d ** -0.5, causal, window, pk, pv), lse)


@pytest.mark.parametrize("window", [None, 40, 1000])
@pytest.mark.parametrize("prefix,parts", [(0, 0), (150, 1), (512, 1), (2100, 5)])
@pytest.mark.parametrize("lens,hq,hk,join_warps", [
    (SEVERAL, 4, 2, 1), (SEVERAL, 10, 2, 1), (SEVERAL, 3, 3, 1), (LONG, 4, 2, 8), (LONG, 32, 2, 8), (SHORT, 4, 2, 1),
    (MANY, 4, 2, 1), ((MANY[0][:2] + (0,) * 19, (2500, 4000) + (1,) * 19), 4, 2, 1)])
def test_heads_of_64(lens, hq, hk, join_warps, prefix, parts, window):
    if prefix and sum(lens[1]) < 4096:
        lens = (lens[0], (lens[1][0] + 4096,) + lens[1][1:])
    run(*lens, hq, hk, 64, "fp16" if hk == 3 else "bf16", prefix, window, parts, join_warps, hq + prefix)


@pytest.mark.parametrize("lens,hq,hk,join_warps", [
    (((1, 2, 0), (20000, 13000, 40)), 4, 1, 8), (((1,) * 40, tuple(500 + 37 * i for i in range(40))), 4, 2, 1),
    (((17, 1) + (0,) * 16, (30000, 3000) + (2,) * 16), 2, 2, None)])
@pytest.mark.parametrize("prefix,parts,window", [(700, 2, None), (3000, 6, 900), (90, 1, 5000)])
def test_heads_of_128_behind_a_prefix(lens, hq, hk, join_warps, prefix, parts, window):
    run(*lens, hq, hk, 128, "bf16", prefix, window, parts, join_warps, prefix)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("lens,hq,hk,join_warps", [(SEVERAL, 4, 2, 1), (SEVERAL, 16, 2, 1), (LONG, 8, 1, 8), (MANY, 2, 1, 1)])
def test_own_keys_alone(lens, hq, hk, join_warps, d):
    for window in (None, 70):
        run(*lens, hq, hk, d, "bf16" if d == 256 else "fp16", 0, window, 0, join_warps, d)
    run(*lens, hq, hk, d, "bf16", 0, None, 0, join_warps, d, causal=False)


@pytest.mark.parametrize("d,prefix,parts", [(64, 0, 0), (128, 0, 0), (256, 0, 0), (64, 700, 2)])
@pytest.mark.parametrize("hq,hk", [(4, 2), (3, 3), (32, 2)])
@pytest.mark.parametrize("window", [None, 65])
def test_unused_slots(d, prefix, parts, hq, hk, window):
    """A batch with unused slots: sequences of many rows, one with more rows than its units take (the rest one by one), one with
    rows but no keys, between steps of one token."""
    q_lens = (1, 23, 0, 40, 1, 5, 30) + (0,) * 93
    k_lens = (500, 1700, 9, 70, 1900, 0, 45) + (0,) * 92 + (3,)
    run(q_lens, k_lens, hq, hk, d, "bf16", prefix, window, parts, 1, d + hq)
    run(q_lens, k_lens, hq, hk, d, "fp16", prefix, None, parts, 1, d + hq, causal=False)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window", [None, 1200])
@pytest.mark.parametrize("d,prefix", [(64, 0), (128, 0), (256, 0), (64, 300), (64, 2100)])
def test_values_that_a_row_does_not_see(d, prefix, window, bad):
    """The last key of sequences of two rows, which the first of them does not see, keys before a window, a whole sequence, and
    what stands behind the last one: the first rows are done again from what they see."""
    import reax_engine_b200 as R
    q_lens, k_lens = (2, 1, 2, 0, 0), (1500, 300, 2600, 4, 100)
    cq, ck = cu(q_lens), cu(k_lens)
    assert plan(cq[-1], ck[-1], 5, 4, 2, d, prefix).few
    q, k, v, pk, pv = tensors(cq[-1], ck[-1] + 50, 4, 2, d, "bf16", d, prefix=prefix)
    ref = reference(q, k, v, cq, ck, d ** -0.5, window=window, prefix_k=pk, prefix_v=pv)
    k, v = k.clone(), v.clone()
    for t in (k, v):
        t[ck[1] - 1] = bad                     # seen by row 1 alone
        t[ck[1]:ck[2]] = bad                   # the whole second sequence
        if window:
            t[ck[2]:ck[3] - window - 1] = bad  # before the windows of rows 3 and 4
        t[ck[3] - 1, 1] = bad                  # of one KV head: row 4 alone, heads 2 and 3
        t[ck[3]:] = bad                        # of sequences without rows, and behind the last
    out = torch.full_like(q, 2.0)
    args = (q, k, v, pk, pv) if prefix else (q, k, v)
    call = R.shared_prefix_attention if prefix else R.prompt_attention
    _, lse = call(*args, dev(cq), dev(ck), window=window, return_lse=True, out=out)
    keep = torch.tensor([[1, 1, 1, 1], [0, 0, 0, 0], [0, 0, 0, 0], [1, 1, 1, 1], [1, 1, 0, 0]], dtype=torch.bool)
    check(out.cpu()[keep], [r[keep] for r in ref], lse.cpu()[keep])
    if bad != -float("inf"):                   # a key of -inf may have weight 0
        assert not torch.isfinite(out.float().cpu()[~keep]).all(-1).any()


def test_a_captured_step_follows_new_lengths():
    """A step behind a prefix captured once, replayed with other lengths: one row a sequence, rows gathered in a few sequences,
    and one sequence with more rows than a unit takes."""
    import reax_engine_b200 as R
    seqs, nk, prefix = 30, 6000, 700
    q, k, v, pk, pv = tensors(seqs, nk, 4, 2, 64, "bf16", 8, prefix=prefix)
    assert plan(seqs, nk, seqs, 4, 2, 64, prefix).few
    cq, ck, out = dev(list(range(seqs + 1))), dev([nk * i // seqs for i in range(seqs + 1)]), torch.zeros_like(q)
    call = lambda: R.shared_prefix_attention(q, k, v, pk, pv, cq, ck, out=out)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for a, b in ((list(range(seqs + 1)), [0] + [nk] * seqs), ([0, 5, 5, 9] + [9] * 26 + [12], [0, 100, 3000] + [5000] * 28),
                 ([0, 24] + [30] * 29, [0, 2500] + [6000] * 29), ([0] * 30 + [2], [0] * 30 + [nk])):
        cq.copy_(dev(a)), ck.copy_(dev(b))
        out.fill_(4.0)
        graph.replay()
        n = a[-1]
        check(out[:n], [x[:n] for x in reference(q[:n], k, v, a, b, 0.125, prefix_k=pk, prefix_v=pv)])
        assert (out[n:] == 4).all()
