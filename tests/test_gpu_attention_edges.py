"""Calls of prompt_attention and shared_prefix_attention at their edges. Tolerances: those of test_gpu_attention."""
import pytest
import torch

from test_gpu_attention import check, cu, dev, reference, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,prefix,keys", [(64, 0, 300), (128, 0, 300), (64, 150, 5000), (256, 150, 300)])
def test_lengths_that_do_not_rise_from_zero(d, prefix, keys):
    """Rows before the first sequence's, and lengths that fall: outside the contract, their values are anything, but rows of
    sequences that are well-formed are right, and so is the next call."""
    import reax_engine_b200 as R
    q, k, v, pk, pv = tensors(12, keys, 4, 2, d, "bf16", d, prefix=prefix)
    call = lambda cq, ck: (R.shared_prefix_attention(q, k, v, pk, pv, dev(cq), dev(ck)) if prefix  # noqa: E731
                           else R.prompt_attention(q, k, v, dev(cq), dev(ck)))
    ck = [0, 40, 100, keys - 20] + [keys] * 10
    cq = [9, 10, 11, 12] + [12] * 10
    ref = reference(q, k, v, cq, ck, d ** -0.5, prefix_k=pk, prefix_v=pv)
    check(call(cq, ck)[9:], [x[9:] for x in ref])
    for bad in ([7, 3, 9, 1, 12] + [12] * 9, [2 ** 31 - 1] * 13 + [12], [-2 ** 31] * 13 + [12], [0] * 13 + [2 ** 31 - 1]):
        call(bad, ck)
        call(cq, [keys - 1, -5, 2 ** 31 - 1, 3] + [-2 ** 31, 7] * 5)
    check(call(cq, ck)[9:], [x[9:] for x in ref])


def test_row_sums_keep_all_their_bits():
    """Weights 1 and 2^-23 (scale ln 2, whose product with log2(e) is 1 in fp32) of values 1 and 12288: the sum of the products is
    1 + 3 2^-11, half-way between two fp16 values, and the sum of the weights, 1 + 2^-23, decides that the lower one is nearer."""
    import math
    import reax_engine_b200 as R
    q, k, v = (torch.zeros(2, 1, 64, dtype=torch.float16, device="cuda") for _ in range(3))
    q[..., 0] = 1
    k[1, 0, 0] = -23
    v[0], v[1] = 1, 12288
    for first in (0, 1):                     # either key first: the halves of the columns add up in another order
        kk, vv = (k, v) if first == 0 else (k.flip(0), v.flip(0))
        o = R.prompt_attention(q, kk, vv, dev([0, 2]), causal=False, scale=math.log(2))
        assert (o == 1 + 2.0 ** -10).all()


def test_an_empty_batch_into_an_output():
    import reax_engine_b200 as R
    q, k, v, pk, pv = tensors(0, 0, 4, 2, 64, "bf16", 1, prefix=5)
    out = torch.empty_like(q)
    assert R.prompt_attention(q, k, v, dev([0, 0]), out=out) is out
    assert R.shared_prefix_attention(q, k, v, pk, pv, dev([0]), out=out) is out


def test_options_that_are_written_in_place():
    """Options given as tensors count with what they hold at the call."""
    import reax_engine_b200 as R
    q, k, v, _, _ = tensors(40, 40, 4, 2, 64, "bf16", 5)
    c = dev([0, 40])
    window, causal, scale = torch.tensor(3), torch.tensor(True), torch.tensor(0.125)
    for w, cs, s in ((3, True, 0.125), (20, True, 0.125), (20, True, 0.5), (3, True, 0.125)):
        window.fill_(w), causal.fill_(cs), scale.fill_(s)
        got = R.prompt_attention(q, k, v, c, window=window, causal=causal, scale=scale)
        assert torch.equal(got, R.prompt_attention(q, k, v, c, window=w, causal=cs, scale=s))
        check(got, reference(q, k, v, [0, 40], [0, 40], s, window=w))
    causal.fill_(False)
    assert torch.equal(R.prompt_attention(q, k, v, c, causal=causal), R.prompt_attention(q, k, v, c, causal=False))
    with pytest.raises(ValueError):
        R.prompt_attention(q, k, v, c, causal=causal, window=window)


def test_tangents_are_refused():
    import reax_engine_b200 as R
    from torch.autograd import forward_ad
    q, k, v, pk, pv = tensors(8, 8, 4, 2, 64, "bf16", 2, prefix=4)
    c = dev([0, 8])
    R.shared_prefix_attention(q, k, v, pk, pv, c)            # (checked calls are remembered)
    with forward_ad.dual_level():
        for i in range(5):
            ts = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate((q, k, v, pk, pv))]
            with pytest.raises(ValueError):
                R.shared_prefix_attention(*ts, c)
        R.shared_prefix_attention(q, k, v, pk, pv, c)


@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16"), (256, "fp16")])
@pytest.mark.parametrize("window", [None, 150])
@pytest.mark.parametrize("prefix", [0, 90])
def test_single_values_that_are_not_finite(d, dtype, window, prefix):
    """Infinities and NaN strewn over single elements of the values: exactly those elements of the outputs are not finite whose
    row sees one there, the others are what they are without them."""
    import reax_engine_b200 as R
    lens = (300, 1, 77, 200)
    c = cu(lens)
    q, k, v, pk, pv = tensors(c[-1], c[-1], 4, 2, d, dtype, d, prefix=prefix)
    bad = torch.zeros(v.shape, dtype=torch.bool, device="cuda")
    for key, head, e in ((5, 0, 1), (20, 0, 1), (290, 0, 1), (130, 0, d - 1), (299, 1, 7), (300, 1, 0), (310, 0, 8), (400, 1, d - 2),
                         (577, 0, 3), (378, 1, 33)):
        bad[key, head, e] = True
    bad[150:155, 1] = True
    pbad = torch.zeros(pv.shape, dtype=torch.bool, device="cuda") if prefix else None
    if prefix:
        pbad[3, 0, 2] = pbad[88, 1, 5] = True
    # what each row sees: a 0 / 1 product over the masks
    seen = torch.zeros(q.shape, dtype=torch.bool)
    for b in range(len(lens)):
        for i in range(c[b], c[b + 1]):
            col = bad[c[b]:i + 1]
            if prefix:
                col = torch.cat([pbad, col])
            if window:
                col = col[-window:]
            seen[i] = col.any(0).repeat_interleave(2, 0).cpu()
    ref = reference(q, k, v.masked_fill(bad, 0), c, c, d ** -0.5, window=window, prefix_k=pk,
                    prefix_v=pv.masked_fill(pbad, 0) if prefix else None)
    assert seen.any() and not seen.all()
    for x in (float("nan"), float("inf")):
        w, pw = v.masked_fill(bad, x), pv.masked_fill(pbad, x) if prefix else None
        o, lse = (R.shared_prefix_attention(q, k, w, pk, pw, dev(c), window=window, return_lse=True) if prefix
                  else R.prompt_attention(q, k, w, dev(c), window=window, return_lse=True))
        assert torch.equal(~torch.isfinite(o.cpu()), seen)
        check(o.cpu()[~seen], [ref[0][~seen], ref[1], ref[2][~seen], ref[3]])
        check(q, (q.cpu().double(), ref[1], torch.ones_like(ref[2]), ref[3]), lse)


def test_one_infinity_does_not_take_the_prompt_with_it():
    """An infinity that half of the rows see costs a pass over the values, not one per row: it took 140 times the call without it
    (D = 128, 8192 tokens, 0.7 ms), and may not take 30 times."""
    import reax_engine_b200 as R
    n = 8192
    q, k, v, _, _ = tensors(n, n, 32, 8, 128, "fp16", 1)
    c = dev([0, n])
    times = []
    for at in (None, n // 2):
        if at:
            v[at, :, 5] = float("inf")
        R.prompt_attention(q, k, v, c)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        o = R.prompt_attention(q, k, v, c)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    bad = ~torch.isfinite(o)
    assert bad[n // 2:, :, 5].all() and int(bad.sum()) == (n - n // 2) * 32
    assert times[1] < 30 * times[0], times


def launches(f):
    """Names and grids of the kernels that f launches, from a captured graph."""
    from cuda.bindings import driver
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        f()
    ok = lambda r: r[1:] if int(r[0]) == 0 else pytest.fail(str(r[0]))  # noqa: E731
    g = driver.CUgraph(graph.raw_cuda_graph())
    nodes = ok(driver.cuGraphGetNodes(g, ok(driver.cuGraphGetNodes(g))[1]))[0]
    found = []
    for n in nodes:
        if ok(driver.cuGraphNodeGetType(n))[0] == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            p = ok(driver.cuGraphKernelNodeGetParams(n))[0]
            name = ok(driver.cuFuncGetName(p.func))[0] if int(p.func) else ok(driver.cuKernelGetName(p.kern))[0]
            found.append((name.decode(), p.gridDimX))
    return found


@pytest.mark.parametrize("d", [64, 128, 256])
def test_grids_within_the_sm_budget(d):
    import reax_engine_b200 as R
    q, k, v, pk, pv = tensors(200, 40000, 4, 4, d, "bf16", 1, prefix=700)
    step = (dev(list(range(201))), dev([200 * i for i in range(201)]))
    calls = {"step": lambda: R.prompt_attention(q, k, v, *step),
             "step behind a prefix": lambda: R.shared_prefix_attention(q, k, v, pk, pv, *step),
             "prompt": lambda: R.prompt_attention(q, k[:200], v[:200], dev_c)}
    dev_c = dev([0, 200])
    try:
        for budget in (0, 20, 7):
            R.set_sm_budget(budget)
            for name, f in calls.items():
                f()
                grids = [n for k_, n in launches(f) if "pair_kernel" in k_ or "few_kernel" in k_]
                assert grids and all(n <= (budget or 2 * 148) for n in grids), (name, budget, grids)
    finally:
        R.set_sm_budget(0)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q_lens,k_lens,prefix", [((300,), (300,), 0), ((3, 2), (5000, 400), 0), ((1,) * 8, (700,) * 8, 0),
                                                  ((1, 40), (3, 40), 3000), ((1,) * 8, (700,) * 8, 1500)])
def test_values_at_the_end_of_fp16(d, q_lens, k_lens, prefix):
    """An average of values of 65504 is 65504, not infinite, however the weights round (larger and larger scores, so that the
    maximum in use lags)."""
    import reax_engine_b200 as R
    cq, ck = cu(q_lens), cu(k_lens)
    q, k, v, pk, pv = tensors(cq[-1], ck[-1], 4, 2, d, "fp16", d, prefix=prefix)
    q, k = q * 0 + 1, (k * 0.02 + torch.linspace(-3, 6, ck[-1], device="cuda")[:, None, None] / d * 8).half()
    v[:, :, ::2], v[:, :, 1] = 65504, -65504
    if prefix:
        pk = pk * 0.02
        pv[:, :, ::2], pv[:, :, 1] = 65504, -65504
    kw = dict(scale=1.0, return_lse=True)
    o, lse = (R.shared_prefix_attention(q, k, v, pk, pv, dev(cq), dev(ck), **kw) if prefix
              else R.prompt_attention(q, k, v, dev(cq), dev(ck), **kw))
    check(o, reference(q, k, v, cq, ck, 1.0, prefix_k=pk, prefix_v=pv), lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,seqs,n,prefix", [(2, 1, 130, 0), (1, 1, 130, 0), (1, 1, 34, 0), (2, 20, 130, 0), (2, 1, 2000, 0),
                                                (1, 30, 200, 600)])
def test_a_rounded_up_weight_does_not_make_a_value_infinite(d, rows, seqs, n, prefix):
    """A row's last two keys have 2^10 (1 + 0.55 2^-10) times the weight of 16 before them (and the others none), which fp16 rounds
    up by 0.45 2^-10 where these 16 are in an earlier tile, relative to whose maximum the weights are: the products with 65504
    then sum to 65532 times the sum of the weights, nearer to infinity than to 65504."""
    import math
    import reax_engine_b200 as R
    q, k, v = (torch.zeros(m, 1, d, dtype=torch.float16, device="cuda") for m in (rows * seqs, n * seqs, n * seqs))
    pk, pv = (torch.zeros(prefix, 1, d, dtype=torch.float16, device="cuda") for _ in range(2))
    q[..., 0], k[..., 0], pk[..., 0] = 1, -30, -30
    for s in range(seqs):
        e = (s + 1) * n
        k[e - 18:e - 2, 0, 0], k[e - 2:e, 0, 0] = 0, 1
    for t in (v, pv):
        t[..., ::2], t[..., 1] = 65504, -65504
    cq, ck = [rows * i for i in range(seqs + 1)], [n * i for i in range(seqs + 1)]
    scale = (10 + math.log2(1 + 0.55 * 2 ** -10)) * math.log(2)
    o = (R.shared_prefix_attention(q, k, v, pk, pv, dev(cq), dev(ck), scale=scale) if prefix
         else R.prompt_attention(q, k, v, dev(cq), dev(ck), scale=scale))
    check(o, reference(q, k, v, cq, ck, scale, prefix_k=pk if prefix else None, prefix_v=pv if prefix else None))
