"""The attention operators on packed batches: what is measured, in plain torch and through the framework's calls.

Two operators. ``prompt``: attention over packed sequences of different lengths (causal from the end of the keys, grouped
heads, an optional sliding window); a single query row per sequence is the same call. ``prefix``: the same for a batch whose
sequences all continue one shared prefix, whose keys and values are stored once.

Tensors: q [tokens, heads, dim], k / v [key tokens, kv_heads, dim], prefix k / v [prefix, kv_heads, dim]; cumulative lengths
int32 [sequences + 1]. Outputs: o [tokens, heads, dim] in the type of q, and the natural logarithm of the softmax's sum
[tokens, heads] fp32 where a case asks for it.
"""
import math
import random

import torch

own = False

BLOCK = 2048    # query rows of one product of the plain form


def _case(name, op, seqs, q_lens, k_lens=None, prefix=0, heads=16, kv_heads=8, dim=256, dtype="bf16", unit=False, window=0,
          views=False, lse=False, lens=1):
    """q_lens / k_lens: the range that a sequence's lengths are drawn from (k_lens None: as many keys as queries). unit: scores
    are not scaled (normalised heads); else by dim ** -0.5. views: q, k and v are slices of one fused projection's output."""
    return dict(name=name, op=op, seqs=seqs, q_lo=q_lens[0], q_hi=q_lens[1], k_lo=k_lens[0] if k_lens else 0,
                k_hi=k_lens[1] if k_lens else 0, prefix=prefix, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, unit=unit,
                window=window, views=views, lse=lse, lens=lens)


def listed():
    return [
        # one short prompt: a request alone, where latency counts
        _case("one short prompt", "prompt", 1, (37, 37), unit=True),
        # four short prompts packed together (a total of about 500 tokens)
        _case("four short prompts", "prompt", 4, (64, 192), lens=2, views=True, lse=True),
        # a batch of 32 prompts of 256 to 2048 tokens
        _case("prompts", "prompt", 32, (256, 2048), lens=3),
        # a decision batch of 64 prompts through a sliding-window layer, heads normalised
        _case("decision, sliding layer", "prompt", 64, (512, 4096), unit=True, window=1024, lens=4),
        # the same batch through a global layer: the largest case
        _case("decision, global layer", "prompt", 64, (512, 4096), unit=True, lens=4),
        # one long document in fp16, heads of 128 in groups of 4, read from the fused projection
        _case("long document", "prompt", 1, (16411, 16411), heads=32, kv_heads=8, dim=128, dtype="fp16", views=True),
        # one query row per prompt: the last layer of a decision forward, or a step of generation
        _case("last rows", "prompt", 64, (1, 1), (512, 4096), unit=True, lens=5),
        # one token after a long context, groups of 8
        _case("one token, long context", "prompt", 1, (1, 1), (131101, 131101), heads=32, kv_heads=4, dim=128, lse=True),
        # 64 short option texts after one shared instruction
        _case("options", "prefix", 64, (3, 40), prefix=2048, unit=True, lens=6),
        # 64 prompts that share a long context
        _case("shared context", "prefix", 64, (64, 768), prefix=4096, lens=7, lse=True),
        # the same kind of batch through a sliding-window layer: only the first rows still see the prefix
        _case("shared context, sliding layer", "prefix", 48, (100, 900), prefix=1500, unit=True, window=1024, lens=8),
        # one token each of 256 sequences with a few keys of their own after a long prefix, 64-wide ungrouped heads, fp16
        _case("tokens, shared prefix", "prefix", 256, (1, 1), (1, 128), prefix=16383, heads=16, kv_heads=16, dim=64,
              dtype="fp16", lens=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prefix"])
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (12, 4), (8, 8), (10, 2), (32, 4)])
    dim = rng.choice([64, 128, 256, 256])
    single = rng.random() < 0.35
    seqs = _log(rng, 1, 96)
    q_hi = 1 if single else _log(rng, 2, min(3000, 60000 // seqs))
    q_lo = 1 if single else _log(rng, 1, q_hi)
    k = None
    if single or rng.random() < 0.25:
        k_hi = _log(rng, q_hi, q_hi + min(60000, 400000 // seqs) if op == "prompt" else q_hi + 400)
        k = (min(_log(rng, 1, k_hi), k_hi), k_hi)
        k = (max(k[0], q_hi), max(k[1], q_hi))
    prefix = 0 if op == "prompt" else _log(rng, 16, 16000 if single else 4000)
    window = rng.choice([0, 0, _log(rng, 2, 4096)])
    return dict({n: v for n, v in _case(
        "", op, seqs, (q_lo, q_hi), k, prefix, heads, kv_heads, dim, rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.5,
        window, k is None and rng.random() < 0.5, rng.random() < 0.5, rng.randrange(1 << 20)).items() if n != "name"})


def _lens(case):
    r = random.Random(case["lens"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
    k = [r.randint(case["k_lo"], case["k_hi"]) for _ in q] if case["k_hi"] else list(q)
    return q, k


def _scale(case):
    return 1.0 if case["unit"] else case["dim"] ** -0.5


def prepare(case, seed):
    """Normal heads. Unscaled scores come from normalised heads whose learned weights keep the scores a few units wide."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float16
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    ql, kl = _lens(case)
    nq, nk = sum(ql), sum(kl)
    amp = 1.6 * d ** -0.25 if case["unit"] else 1.5      # of q and k: their products have a spread of about 2.4

    def heads(n, h, s):
        return (torch.randn(n, h, d, generator=g, device="cuda") * s).to(dt)

    if case["views"]:
        qkv = torch.cat([heads(nq, hq + hk, amp), heads(nq, hk, 1.0)], 1)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    else:
        q, k, v = heads(nq, hq, amp), heads(nk, hk, amp), heads(nk, hk, 1.0)
    cu_q = torch.tensor([0] + ql).cumsum(0).to(torch.int32).cuda()
    cu_k = torch.tensor([0] + kl).cumsum(0).to(torch.int32).cuda()
    state = dict(case=case, q=q, k=k, v=v, cu_q=cu_q, cu_k=cu_k, q_lens=ql, k_lens=kl)
    if case["op"] == "prefix":
        state.update(prefix_k=heads(case["prefix"], hk, amp), prefix_v=heads(case["prefix"], hk, 1.0))
    return state


def _plain(state):
    case, q = state["case"], state["q"]
    hk, prefix, window, scale = case["kv_heads"], case["prefix"], case["window"], _scale(case)
    group = case["heads"] // hk
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    if prefix:
        pk, pv = state["prefix_k"].float().transpose(0, 1), state["prefix_v"].float().transpose(0, 1)
    a = b = 0
    for m, n in zip(state["q_lens"], state["k_lens"]):
        kk, vv = state["k"][b:b + n].float().transpose(0, 1), state["v"][b:b + n].float().transpose(0, 1)
        if prefix:
            kk, vv = torch.cat([pk, kk], 1), torch.cat([pv, vv], 1)
        first = prefix + n - m                           # position of the sequence's first query row
        for i in range(0, m, BLOCK):
            rows = min(BLOCK, m - i)
            hi = first + i + rows                        # no later key is seen by these rows
            lo = max(0, first + i - window + 1) if window else 0
            qq = q[a + i:a + i + rows].float().reshape(rows, hk, group, -1).permute(1, 2, 0, 3).reshape(hk, group * rows, -1)
            s = (qq @ kk[:, lo:hi].transpose(1, 2)).mul_(scale).view(hk, group, rows, hi - lo)
            pos = torch.arange(first + i, first + i + rows, device=q.device)[:, None]
            j = torch.arange(lo, hi, device=q.device)[None, :]
            masked = j > pos
            if window:
                masked = masked | (j <= pos - window)
            s.masked_fill_(masked, float("-inf"))
            top = s.amax(-1, keepdim=True)
            s.sub_(top).exp_()
            total = s.sum(-1, keepdim=True)
            o = (s.view(hk, group * rows, hi - lo) @ vv[:, lo:hi]).view(hk, group, rows, -1) / total
            out[a + i:a + i + rows] = o.permute(2, 0, 1, 3).reshape(rows, hk * group, -1).to(q.dtype)
            lse[a + i:a + i + rows] = (top + total.log()).squeeze(-1).permute(2, 0, 1).reshape(rows, -1)
        a, b = a + m, b + n
    return {"o": out, "lse": lse} if case["lse"] else {"o": out}


def run(state):
    if not own:
        return _plain(state)
    import reax_engine_b200 as R
    case = state["case"]
    kw = dict(scale=_scale(case), window=case["window"] or None, return_lse=case["lse"])
    if case["op"] == "prompt":
        r = R.prompt_attention(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], **kw)
    else:
        r = R.shared_prefix_attention(state["q"], state["k"], state["v"], state["prefix_k"], state["prefix_v"], state["cu_q"],
                                      state["cu_k"], **kw)
    return {"o": r[0], "lse": r[1]} if case["lse"] else {"o": r}


def work(case):
    """Each query row, output row and key that some row sees once; 4 * dim operations for each pair of a row and a key."""
    d, w, p = case["dim"], case["window"], case["prefix"]
    pairs = own_keys = 0
    prefix_from = p
    for m, n in zip(*_lens(case)):
        first = p + n - m
        last = first + m - 1
        if not w:
            pairs += m * (first + 1) + m * (m - 1) // 2
            own_keys, prefix_from = own_keys + n, 0
        else:
            full = max(0, min(m, last - max(first, w - 1) + 1))    # rows that see w keys
            rest = m - full                                        # the rows before them see all keys up to their own
            pairs += full * w + rest * (first + 1) + rest * (rest - 1) // 2
            seen_from = max(0, first - w + 1)
            own_keys += last + 1 - max(p, seen_from)
            prefix_from = min(prefix_from, seen_from)
    ql, _ = _lens(case)
    nq, hq, hk = sum(ql), case["heads"], case["kv_heads"]
    size = 2 * d * (2 * nq * hq + 2 * (own_keys + p - prefix_from) * hk)
    return {"bytes": size + (4 * nq * hq if case["lse"] else 0) + 8 * (case["seqs"] + 1), "flops": 4 * d * hq * pairs}


def exact(case, seed):
    """By the definition, in 64 bits, head by head: weights exp(s - max) over the keys a row may see."""
    state = prepare(case, seed)
    dev = state["q"].device
    q, k, v = state["q"], state["k"], state["v"]
    p, w, group = case["prefix"], case["window"], case["heads"] // case["kv_heads"]
    o = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=dev)
    q_at = k_at = 0
    for m, n in zip(state["q_lens"], state["k_lens"]):
        for kv in range(case["kv_heads"]):
            keys, values = k[k_at:k_at + n, kv].double(), v[k_at:k_at + n, kv].double()
            if p:
                keys = torch.vstack([state["prefix_k"][:, kv].double(), keys])
                values = torch.vstack([state["prefix_v"][:, kv].double(), values])
            index = torch.arange(p + n, device=dev)
            for r0 in range(0, m, 4096):
                r1 = min(m, r0 + 4096)
                at = p + n - m + torch.arange(r0, r1, device=dev)
                seen = index <= at.unsqueeze(1)
                if w:
                    seen &= index > at.unsqueeze(1) - w
                for h in range(kv * group, (kv + 1) * group):
                    s = _scale(case) * torch.einsum("id,jd->ij", q[q_at + r0:q_at + r1, h].double(), keys)
                    s = torch.where(seen, s, -torch.inf)
                    lse[q_at + r0:q_at + r1, h] = torch.logsumexp(s, 1)
                    o[q_at + r0:q_at + r1, h] = torch.softmax(s, 1) @ values
        q_at, k_at = q_at + m, k_at + n
    return {"o": o, "lse": lse} if case["lse"] else {"o": o}
