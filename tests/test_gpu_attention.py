"""prompt_attention and shared_prefix_attention against the definition in 64 bits.

Tolerances, from the arithmetic. With u = eps / 2 of the operands' type (bf16 2^-8, fp16 2^-11) and A = sum_j w_j |v_j| for the
softmax weights w:
  * the weights are rounded to the operands' type before the second product: at most u A;
  * the output is rounded once: at most u |o| (and half of the smallest subnormal);
  * a score is a sum of d products in fp32, each addition off by at most 2^-23 of the running magnitude:
    e = d 2^-23 scale max_j sum |q k_j|; its weight moves by e relative, and so does the sum that divides: 2 e A;
  * scaling, subtraction of the maximum, exp2, the sums over keys and the division in fp32: 2^-18 A covers them, and the score's
    scaling in units of log2 adds 2^-22 max|s| A.
lse: e + 2^-22 max|s| + 2^-18.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": (torch.bfloat16, 2.0 ** -8, 0.0), "fp16": (torch.float16, 2.0 ** -11, 2.0 ** -25)}


def reference(q, k, v, cu_q, cu_k, scale, causal=True, window=None, prefix_k=None, prefix_v=None):
    """o, lse, and the tolerances of both, [tokens, heads, ...] in 64 bits on the CPU, key by key as defined."""
    u, tiny = next((x[1], x[2]) for x in DT.values() if x[0] == q.dtype)
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    P = 0 if prefix_k is None else prefix_k.shape[0]
    g, d = q.shape[1] // k.shape[1], q.shape[2]
    o = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -torch.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64)
    for b in range(len(cu_q) - 1):
        for i in range(cu_q[b], cu_q[b + 1]):
            kk, vv = k[cu_k[b]:cu_k[b + 1]], v[cu_k[b]:cu_k[b + 1]]
            if P:
                kk, vv = torch.cat([prefix_k.cpu().double(), kk]), torch.cat([prefix_v.cpu().double(), vv])
            n, t = kk.shape[0], kk.shape[0] - (cu_q[b + 1] - i)
            hi = min(max(t + 1, 0), n) if causal else n
            lo = max(0, t - window + 1) if window else 0
            if hi <= lo:
                continue
            kk = kk[lo:hi].repeat_interleave(g, 1)
            vv = vv[lo:hi].repeat_interleave(g, 1)
            s = scale * torch.einsum("hd,jhd->hj", q[i], kk)
            w = s.softmax(-1)
            o[i] = torch.einsum("hj,jhd->hd", w, vv)
            lse[i] = s.logsumexp(-1)
            e = d * 2.0 ** -23 * scale * torch.einsum("hd,jhd->hj", q[i].abs(), kk.abs()).amax(-1) + 2.0 ** -22 * s.abs().amax(-1)
            big = torch.einsum("hj,jhd->hd", w, vv.abs())
            tol[i] = u * o[i].abs() + (u + 2 * e + 2.0 ** -18)[:, None] * big + tiny
            ltol[i] = e + 2.0 ** -18
    return o, lse, tol, ltol


def cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return c


def tensors(nq, nk, hq, hk, d, dtype, seed, prefix=0, amp=1.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = lambda n, h, s=1.0: (torch.randn(n, h, d, generator=g, device="cuda") * s).to(DT[dtype][0])  # noqa: E731
    r = [t(nq, hq, amp), t(nk, hk, amp), t(nk, hk)]
    return r + ([t(prefix, hk, amp), t(prefix, hk)] if prefix else [None, None])


def dev(c, dtype=torch.int32):
    return torch.tensor(c, dtype=dtype, device="cuda")


def check(got, ref, lse=None):
    o, l, tol, ltol = ref
    got = got.detach().cpu().double()
    bad = (got - o).abs() > tol
    assert not (bad | ~torch.isfinite(got)).any(), \
        f"{int(bad.sum())} of {bad.numel()} off; worst {((got - o).abs() / (tol + 1e-300)).max():.2f} of the tolerance"
    if lse is not None:
        x = lse.cpu().double()
        none = torch.isinf(l)
        assert torch.equal(x[none], l[none]) and ((x - l).abs()[~none] <= ltol[~none]).all()


def run(q_lens, k_lens=None, hq=4, hk=2, d=64, dtype="bf16", causal=True, window=None, prefix=0, seed=0, scale=None):
    import reax_engine_b200 as R
    cq, ck = cu(q_lens), cu(k_lens or q_lens)
    q, k, v, pk, pv = tensors(cq[-1], ck[-1], hq, hk, d, dtype, seed, prefix)
    kw = dict(scale=scale, causal=causal, window=window, return_lse=True)
    args = (dev(cq), None if k_lens is None else dev(ck))
    o, lse = (R.shared_prefix_attention(q, k, v, pk, pv, *args, **kw) if prefix else R.prompt_attention(q, k, v, *args, **kw))
    check(o, reference(q, k, v, cq, ck, scale or d ** -0.5, causal, window, pk, pv), lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens", [(1,), (37,), (128,), (129, 1, 0, 127), (300, 5)])
def test_prompts(d, dtype, lens):
    run(lens, d=d, dtype=dtype, seed=sum(lens))


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (6, 2), (5, 1), (14, 2), (16, 1), (96, 2), (128, 1), (77, 1)])
def test_groups_of_heads(hq, hk):
    run((70, 3, 61), hq=hq, hk=hk, d=128, seed=hq)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("window", [1, 2, 63, 128, 200, 10 ** 9])
def test_windows(d, window):
    run((260, 40, 1), d=d, window=window, seed=window % 97)


@pytest.mark.parametrize("q_lens,k_lens", [
    ((1, 1, 1), (300, 1, 129)),          # single tokens
    ((2, 0, 5), (2, 400, 9)),            # keys of a sequence without query rows lie between
    ((4, 3, 2), (1, 0, 2)),              # rows that see nothing: more query rows than keys, and no keys at all
    ((40,), (700,)),                     # a chunk of a prompt after its first part
    ((0, 0, 3, 0), (5, 0, 3, 0)),
])
@pytest.mark.parametrize("window", [None, 50])
@pytest.mark.parametrize("d", [64, 256])
def test_other_key_lengths(q_lens, k_lens, window, d):
    run(q_lens, k_lens, d=d, window=window, seed=7)


@pytest.mark.parametrize("d", [64, 128])
def test_every_key(d):
    run((100, 33), (257, 64), d=d, causal=False, seed=3)
    run((20, 33), (57, 0), d=d, causal=False, seed=4)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("prefix", [1, 128, 331])
@pytest.mark.parametrize("q_lens,k_lens,window", [
    ((3, 40, 1, 0, 130), None, None), ((1,) * 20, (1, 5, 0, 9) * 5, None), ((30, 200, 2), None, 64), ((3, 9), (1, 9), None),
    ((1,) * 12, (200, 3, 1) * 4, 100)])
def test_shared_prefix(d, prefix, q_lens, k_lens, window):
    run(q_lens, k_lens, d=d, prefix=prefix, window=window, seed=prefix + d)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prefix_alone_without_own_keys(dtype):
    run((2, 5), (0, 0), d=128, dtype=dtype, prefix=140)


def test_many_rows_split_and_whole_agree():
    """Long keys with few rows are split over the keys and joined; the same rows in a larger batch are not."""
    run((1,), (5000,), hq=8, hk=1, d=128, seed=1)
    run((2, 3), (2600, 3000), hq=2, hk=1, d=64, seed=2)
    run((1, 1), (1, 4000), hq=4, hk=4, d=256, window=3500, seed=3)
    run((1,) * 6, (3,) * 6, hq=4, hk=1, d=256, prefix=3000, seed=4)


def test_more_tiles_than_pairs():
    """More row tiles than CTA pairs, the last of them nearly empty, so that every pair works through several."""
    import reax_engine_b200 as R
    for d, dtype, lens in ((64, "bf16", (700, 1, 0, 900, 401)), (256, "fp16", (1300, 37))):
        c = cu(lens)
        q, k, v, _, _ = tensors(c[-1], c[-1], 16, 16, d, dtype, 6)
        o, lse = R.prompt_attention(q, k, v, dev(c), return_lse=True)
        for h in (0, 9, 15):
            one = [t[:, h:h + 1] for t in (q, k, v)]
            check(o[:, h:h + 1], reference(*one, c, c, d ** -0.5), lse[:, h:h + 1])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q_lens,k_lens,hq,hk", [
    ((1,) * 7, (40, 1, 700, 0, 16, 17, 300), 4, 2),
    ((2, 0, 1, 0, 3), (100, 30, 64, 1, 200), 4, 1),          # several rows of a sequence, others without any
    ((1, 1, 1), (130, 257, 90), 16, 1),                      # 16 rows a sequence
    ((1, 1), (50, 60), 10, 2),
    ((20,) + (0,) * 23, (500,) + (3,) * 23, 4, 2),           # more rows of a sequence than the generation step's kernel takes
    ((1,) * 40, (64,) * 40, 2, 2),
])
@pytest.mark.parametrize("window,prefix", [(None, 0), (33, 0), (None, 150), (90, 40)])
def test_generation_steps(q_lens, k_lens, hq, hk, window, prefix, d):
    run(q_lens, k_lens, hq=hq, hk=hk, d=d, window=window, prefix=prefix, dtype="bf16" if d != 128 else "fp16", seed=len(q_lens) + d)


def test_generation_step_beside_values_that_it_does_not_see():
    import reax_engine_b200 as R
    for d, hq, hk in ((64, 4, 2), (256, 2, 1)):
        cq, ck = [0, 1, 2, 4], [0, 200, 203, 400]
        q, k, v, pk, pv = tensors(6, 450, hq, hk, d, "bf16", d, prefix=70)
        ref = reference(q, k, v, cq, ck, d ** -0.5, window=60, prefix_k=pk, prefix_v=pv)
        k, v = k.clone(), v.clone()
        for t in (k, v):
            t[200:203] = float("nan")      # the whole second sequence
            t[:130] = float("inf")         # before the window
            t[399] = float("-inf")         # after the last row but one
            t[400:] = float("nan")         # behind the last sequence
        out = torch.full_like(q, 2.0)
        _, lse = R.shared_prefix_attention(q, k, v, pk, pv, dev(cq), dev(ck), window=60, out=out, return_lse=True)
        keep = torch.tensor([True, False, True, False])
        check(out[:4].cpu()[keep], [r[:4][keep] for r in ref], lse[:4].cpu()[keep])
        assert (out[4:] == 2).all() and torch.isnan(out[1].float()).any()


def test_large_and_small_scores():
    """Scores of hundreds, whose running maximum grows from tile to tile, and weights far below the largest."""
    import reax_engine_b200 as R
    for dtype in DT:
        q, k, v, _, _ = tensors(300, 300, 2, 1, 128, dtype, 11)
        k = (k.float() * torch.linspace(0.1, 6.0, 300, device="cuda")[:, None, None]).to(k.dtype)   # later keys weigh more
        c = [0, 300]
        for kk in (k, k.flip(0)):
            o, lse = R.prompt_attention(q, kk, v, dev(c), scale=0.7, return_lse=True)
            check(o, reference(q, kk, v, c, c, 0.7), lse)
            o, lse = R.prompt_attention(q[:1], kk, v, dev([0, 1]), dev(c), scale=0.7, return_lse=True)
            check(o, reference(q[:1], kk, v, [0, 1], c, 0.7), lse)
        flat = torch.zeros_like(q)      # every weight the same
        o, lse = R.prompt_attention(flat, k, v, dev(c), return_lse=True)
        check(o, reference(flat, k, v, c, c, 128 ** -0.5), lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_a_row_does_not_see(d, bad):
    """NaN and infinities behind a row's last key, before its window, in other sequences and behind the last one."""
    import reax_engine_b200 as R
    c = [0, 70, 75, 200]
    q, k, v, pk, pv = tensors(210, 210, 4, 2, d, "bf16", 5, prefix=40)
    ref = reference(q, k, v, c, c, d ** -0.5, window=30, prefix_k=pk, prefix_v=pv)
    k, v = k.clone(), v.clone()
    for t in (k, v):
        t[70:75] = bad             # a whole sequence
        t[150, 1] = bad            # one key of one head: rows 150..179 of its query heads see it
        t[200:] = bad              # behind the last sequence
    o, lse = R.shared_prefix_attention(q, k, v, pk, pv, dev(c), window=30, return_lse=True)
    keep = torch.ones(200, 4, dtype=torch.bool)
    keep[70:75] = False
    keep[150:180, 2:] = False
    check(o[:200].cpu()[keep], [r[:200][keep] for r in ref], lse[:200].cpu()[keep])
    want = torch.isnan(o[:200].float().cpu()) | torch.isinf(o[:200].float().cpu())
    if bad != -float("inf"):       # a key of -inf may have weight 0; its value has none of these then
        assert want.any(-1)[~keep].all()


def test_a_query_row_that_is_not_finite_stays_alone():
    import reax_engine_b200 as R
    c = [0, 90, 140]
    q, k, v, _, _ = tensors(140, 140, 2, 2, 128, "fp16", 8)
    ref = reference(q, k, v, c, c, 128 ** -0.5)
    q[17, 1] = float("nan")
    q[100, 0, 3] = float("inf")
    o = R.prompt_attention(q, k, v, dev(c))
    keep = torch.ones(140, 2, dtype=torch.bool)
    keep[17, 1] = keep[100, 0] = False
    check(o.cpu()[keep], [r[keep] for r in ref])
    assert torch.isnan(o[17, 1].float()).all() and torch.isnan(o[100, 0].float()).all()


def test_rows_behind_the_last_sequence_stay():
    import reax_engine_b200 as R
    q, k, v, pk, pv = tensors(300, 300, 4, 2, 64, "bf16", 9, prefix=20)
    c = [0, 100, 170]
    out = torch.full_like(q, 7.0)
    r = R.shared_prefix_attention(q, k, v, pk, pv, dev(c), out=out)
    assert r is out and (out[170:] == 7).all()
    check(out[:170], [x[:170] for x in reference(q, k, v, c, c, 64 ** -0.5, prefix_k=pk, prefix_v=pv)])
    before = out.clone()
    assert R.prompt_attention(q, k, v, dev([0]), out=out) is out and torch.equal(out, before)
    assert R.prompt_attention(q[:0], k[:0], v[:0], dev([0, 0])).shape == (0, 4, 64)
    one = torch.full_like(q, 3.0)
    R.prompt_attention(q, k, v, dev([0, 0, 0]), out=one)
    assert (one == 3).all()


def test_layouts():
    """Slices of one fused projection, heads before tokens, odd offsets, an output with gaps, int64 lengths."""
    import reax_engine_b200 as R
    g = torch.Generator(device="cuda").manual_seed(1)
    n, hq, hk, d = 150, 6, 3, 64
    c = [0, 93, 150]
    qkv = torch.randn(n, hq + 2 * hk, d, generator=g, device="cuda").bfloat16()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    ref = reference(q, k, v, c, c, d ** -0.5)
    check(R.prompt_attention(q, k, v, dev(c, torch.int64)), ref)
    ht = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    check(R.prompt_attention(*ht, dev(c)), ref)
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    check(R.prompt_attention(*odd, dev(c)), ref)
    wide = torch.full((n, hq + 1, 2 * d), 5.0, dtype=q.dtype, device="cuda")
    R.prompt_attention(q, k, v, dev(c), out=wide[:, 1:, d:])
    check(wide[:, 1:, d:], ref)
    assert (wide[:, 0] == 5).all() and (wide[:, :, :d] == 5).all()
    shared = k[:, :1].expand(n, hk, d)                       # one head broadcast to all
    check(R.prompt_attention(q, shared, v, dev(c)), reference(q, shared, v, c, c, d ** -0.5))


def test_same_bits_again_and_under_a_graph():
    """Repeated calls agree bit for bit, on other streams and when captured; two captured graphs do not share a workspace."""
    import reax_engine_b200 as R
    graphs = []
    for seed, (ql, kl) in enumerate([((1,), (4000,)), ((200, 300), (200, 300))]):
        q, k, v, pk, pv = tensors(sum(ql), sum(kl), 4, 2, 128, "bf16", seed, prefix=700)
        cq, ck = dev(cu(ql)), dev(cu(kl))
        want = R.shared_prefix_attention(q, k, v, pk, pv, cq, ck)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = R.shared_prefix_attention(q, k, v, pk, pv, cq, ck)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(want, other)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = R.shared_prefix_attention(q, k, v, pk, pv, cq, ck)
        graphs.append((graph, out, want, (q, k, v, pk, pv, cq, ck)))
    for _ in range(2):
        for graph, out, _, _ in graphs:
            out.zero_()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, (graph, _, _, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in graphs:
            assert torch.equal(out, want)


def test_new_lengths_in_a_captured_call():
    """The cumulative lengths are read on the device: a replay follows what they hold then."""
    import reax_engine_b200 as R
    q, k, v, _, _ = tensors(200, 200, 4, 2, 64, "bf16", 2)
    c = dev([0, 100, 200])
    out = torch.zeros_like(q)
    R.prompt_attention(q, k, v, c, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        R.prompt_attention(q, k, v, c, out=out)
    for lens in ([0, 30, 200], [0, 199, 200], [0, 0, 200]):
        c.copy_(dev(lens))
        graph.replay()
        check(out, reference(q, k, v, lens, lens, 64 ** -0.5))


def test_no_keys_at_all():
    import reax_engine_b200 as R
    q, k, v, pk, pv = tensors(5, 0, 4, 2, 128, "bf16", 1, prefix=3)
    c, ck = dev([0, 2, 5]), dev([0, 0, 0])
    o, lse = R.prompt_attention(q, k, v, c, ck, return_lse=True)
    assert (o == 0).all() and (lse == -torch.inf).all()
    o, lse = R.shared_prefix_attention(q, k, v, pk[:0], pv[:0], c, ck, return_lse=True)
    assert (o == 0).all() and (lse == -torch.inf).all()
    o, lse = R.shared_prefix_attention(q, k, v, pk, pv, c, ck, causal=False, return_lse=True)
    check(o, reference(q, k, v, [0, 2, 5], [0, 0, 0], 128 ** -0.5, causal=False, prefix_k=pk, prefix_v=pv), lse)


@pytest.mark.parametrize("rows", [1, 40])
def test_offsets_past_32_bits(rows):
    """Keys behind the 2^31st element of their buffer (whose rest holds whatever memory held), query and output rows 2^22 elements
    apart."""
    import reax_engine_b200 as R
    n, hk, d, tail = 1_100_000, 8, 256, 300
    k, v = (torch.empty(n, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q0, k0, v0, _, _ = tensors(rows, tail, 16, hk, d, "bf16", 3)
    k[-tail:], v[-tail:] = k0, v0
    span = (600 - 1) * (1 << 22) + 16 * d
    q, out = (torch.empty(span, dtype=torch.bfloat16, device="cuda").as_strided((600, 16, d), (1 << 22, d, 1)) for _ in range(2))
    q[-rows:] = q0
    ck = [0, n - tail, n]
    o, lse = R.prompt_attention(q[600 - rows:], k, v, dev([0, 0, rows]), dev(ck), out=out[600 - rows:], return_lse=True)
    check(o, reference(q0, k0, v0, [0, rows], [0, tail], d ** -0.5), lse)


def test_first_call_of_a_process_under_capture():
    code = (
        "import torch, reax_engine_b200 as R\n"
        "t = [torch.randn(30, h, 64, device='cuda').bfloat16() for h in (4, 2, 2)]\n"
        "c = torch.tensor([0, 10, 30], dtype=torch.int32, device='cuda')\n"
        "torch.cuda.synchronize()\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    o = R.prompt_attention(*t, c)\n"
        "g.replay()\n"
        "torch.cuda.synchronize()\n"
        "assert torch.equal(o, R.prompt_attention(*t, c)) and o.float().abs().sum() > 0\n")
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_sm_budget():
    """Fewer SMs, other parts of the keys: the same answers, and workspaces of the new sizes."""
    import reax_engine_b200 as R
    q, k, v, pk, pv = tensors(3, 3000, 4, 1, 64, "bf16", 4, prefix=1000)
    cq, ck = [0, 1, 2, 3], [0, 1500, 1503, 3000]
    ref = reference(q, k, v, cq, ck, 64 ** -0.5, prefix_k=pk, prefix_v=pv)
    try:
        for sms in (1, 20, 0, 75):
            R.set_sm_budget(sms)
            check(R.shared_prefix_attention(q, k, v, pk, pv, dev(cq), dev(ck)), ref)
            check(R.prompt_attention(q, k, v, dev(cq), dev(ck)), reference(q, k, v, cq, ck, 64 ** -0.5))
    finally:
        R.set_sm_budget(0)


def test_workspace_and_status():
    import reax_engine_b200 as R
    from reax_engine_b200 import _lib as L
    q, k, v, _, _ = tensors(1, 4000, 8, 1, 64, "bf16", 2)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = R.prompt_attention(q, k, v, dev([0, 1]), dev([0, 4000]), workspace=ws, status=status)
    assert torch.equal(a, R.prompt_attention(q, k, v, dev([0, 1]), dev([0, 4000]))) and int(status) == 0
    with pytest.raises(L.ReaxMoEError) as e:
        R.prompt_attention(q, k, v, dev([0, 1]), dev([0, 4000]), workspace=ws[:64])
    assert e.value.code == L.ERR_WORKSPACE


def test_refusals_on_device_tensors():
    import reax_engine_b200 as R
    q, k, v, pk, pv = tensors(8, 8, 4, 2, 64, "bf16", 2, prefix=4)
    c = dev([0, 8])
    bad = [
        lambda: R.prompt_attention(q.float(), k.float(), v.float(), c),
        lambda: R.prompt_attention(q, k.half(), v, c),
        lambda: R.prompt_attention(q, k, v[:7], c),
        lambda: R.prompt_attention(q, k[:, :1], v, c),
        lambda: R.prompt_attention(q[:, :3], k, v, c),
        lambda: R.prompt_attention(q[..., :32], k[..., :32], v[..., :32], c),
        lambda: R.prompt_attention(q, k, v, c, window=0),
        lambda: R.prompt_attention(q, k, v, c, window=4, causal=False),
        lambda: R.prompt_attention(q, k, v, c, scale=0.0),
        lambda: R.prompt_attention(q, k, v, c, scale=float("inf")),
        lambda: R.prompt_attention(q, k, v, c.float()),
        lambda: R.prompt_attention(q, k, v, c, dev([0, 4, 8])),
        lambda: R.prompt_attention(q, k, v, c.cpu()),
        lambda: R.prompt_attention(q, k, v, c, out=q),
        lambda: R.prompt_attention(q, k, v, c, out=q[:4]),
        lambda: R.prompt_attention(q[0], k, v, c),
        lambda: R.prompt_attention(q.clone().requires_grad_(), k, v, c),
        lambda: R.shared_prefix_attention(q, k, v, pk, pv[:3], c),
        lambda: R.shared_prefix_attention(q, k, v, pk[:, :1], pv[:, :1], c),
    ]
    for f in bad:
        with pytest.raises((ValueError, RuntimeError)):
            f()
    with torch.no_grad():
        R.prompt_attention(q.clone().requires_grad_(), k, v, c)
