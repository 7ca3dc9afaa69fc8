"""The index arithmetic of a generation step's kernels (attention_rows.cuh, attention_few.cuh) restated, over cumulative lengths
that hold anything: rows, keys and partial results stay inside their tensors."""
import random

import pytest

ROWS = 16


def int32(x):
    assert -2 ** 31 <= x < 2 ** 31, "overflows an int"
    return x


def sequence_by_warp(is_left, seqs):
    b0, n = 0, seqs
    while n > 1:
        step = (n + 31) // 32
        c = max(sum(lane * step < n and is_left(b0 + lane * step) for lane in range(32)), 1) - 1
        b0 += min(c * step, n - 1)
        n = max(min(step, n - c * step), 1)
    assert 0 <= b0 < seqs
    return b0


def sequence_at(cu_q, cu_k, b, prefix, k_tokens, q_tokens):
    ks = min(max(cu_k[b], 0), k_tokens)
    return ks, prefix + min(max(cu_k[b + 1], ks), k_tokens) - ks, min(max(cu_q[b + 1], 0), q_tokens)


def row_keys_in(s, t, prefix, k_tokens, causal, window):
    ks, everything, q_end = s
    pos = int32(everything - max(int32(q_end - t), 1))
    hi = min(max(pos, -1) + 1, everything) if causal else everything
    lo = min(pos - window + 1, hi) if window > 0 and pos >= window else 0
    p_lo, p_hi, k_lo, k_hi = min(lo, prefix), min(hi, prefix), ks + max(lo - prefix, 0), ks + max(hi - prefix, 0)
    assert 0 <= p_lo <= p_hi <= prefix and 0 <= k_lo <= k_hi <= k_tokens
    return k_lo, k_hi


def lengths(rng, kind, seqs, n):
    some = {"rising": lambda: rng.randint(0, n), "any": lambda: rng.randint(0, n), "past the ends": lambda: rng.randint(-5, n + 9),
            "wild": lambda: rng.choice([0, 1, -1, -2 ** 31, 2 ** 31 - 1, rng.randint(0, n)])}[kind]
    r = [some() for _ in range(seqs + 1)]
    return r if kind in ("any", "wild") else sorted(r)


@pytest.mark.parametrize("kind", ["rising", "any", "past the ends", "wild"])
def test_generation_step_stays_inside(kind):
    rng = random.Random(kind)
    for _ in range(500):
        seqs, q_tokens, k_tokens = rng.randint(1, 70), rng.randint(1, 60), rng.randint(1, 300)
        prefix, group, chunk = rng.choice([0, 0, 7]), rng.choice([1, 2, 5, 16]), rng.choice([64, 80])
        causal = rng.random() < 0.8
        window = rng.choice([0, 1, 30]) if causal else 0
        cu_q, cu_k = lengths(rng, kind, seqs, q_tokens), lengths(rng, kind, seqs, k_tokens)
        units, ntok = -(-k_tokens // chunk) + seqs, min(cu_q[seqs], q_tokens)
        at = lambda b: sequence_at(cu_q, cu_k, b, prefix, k_tokens, q_tokens)  # noqa: E731
        keys = lambda s, t: row_keys_in(s, t, prefix, k_tokens, causal, window)  # noqa: E731
        done = {}                                             # first row of a unit's 16 (by sequence), its keys: by unit
        for u in range(units):                                # find_unit
            b = sequence_by_warp(lambda i: min(max(cu_k[i], 0), k_tokens) // chunk + i <= u, seqs)
            s, c = at(b), u - b
            q0, q1, ke = max(cu_q[b], 0), min(s[2], ntok), s[0] + s[1] - prefix
            if s[0] >= ke or not s[0] // chunk <= c <= (ke - 1) // chunk or q0 >= q1:
                continue
            total = (q1 - q0) * group
            row0 = (c - s[0] // chunk) * ROWS if total > ROWS else 0
            if row0 >= total:
                continue
            rows = min(total - row0, ROWS)
            token = lambda r: q0 + (row0 + min(r, rows - 1)) // group  # noqa: E731
            assert q0 <= token(0) <= token(ROWS) < q1 <= q_tokens
            first, last = keys(s, token(0))[0], keys(s, token(ROWS))[1]
            if total <= ROWS:
                first, last = max(c * chunk, first), min((c + 1) * chunk, last)
            assert first >= last or 0 <= first < last <= k_tokens
            done[u] = b, row0, rows, first, last
        for tok in range(ntok):                               # join_kernel
            b = sequence_by_warp(lambda i: cu_q[i] <= tok, seqs)
            s = at(b)
            k_lo, k_hi = keys(s, tok)
            q0, q1, ke = max(cu_q[b], 0), min(s[2], ntok), s[0] + s[1] - prefix
            if tok < q0 or tok >= q1:
                continue                                      # a row by itself (row_by_warp)
            first, n = s[0] // chunk + b, (ke - 1) // chunk - s[0] // chunk + 1 if s[0] < ke else 0
            by_rows = (q1 - q0) * group > ROWS
            for row in range((tok - q0) * group, (tok - q0 + 1) * group):
                if by_rows and n > 0 and row // ROWS >= n:
                    continue                                  # likewise
                unit = first + (row // ROWS if by_rows else 0)
                own = range(unit, unit + (min(n, 1) if by_rows else n))
                assert all(0 <= u < units for u in own) and (row % ROWS == row or by_rows)
                if kind == "rising":                          # every result was left, and together they have the row's keys
                    got = []
                    for u in own:
                        assert done[u][0] == b and 0 <= row - done[u][1] < done[u][2]
                        got += range(max(done[u][3], k_lo), min(done[u][4], k_hi))
                    assert got == list(range(k_lo, k_hi))
        for t in (0, q_tokens, 2 ** 31 - 1):                  # what the loader may ask for
            keys(at(rng.randrange(seqs)), t)
