"""How reaxmoe_attention divides a call's work, restated: which kernels a call runs shows only in its workspace's size, and with
this a test can say which ones its cases are meant for (a rule that moves fails there, not silently)."""
from dataclasses import dataclass

SMS = 148


@dataclass
class Plan:
    few: bool        # a generation step: few_kernel and join_kernel, after pair_kernel for a prefix
    parts: int       # of the keys that pair_kernel goes over
    join_warps: int  # of join_kernel, a row
    workspace: int


def plan(q_tokens, k_tokens, seqs, q_heads, kv_heads, d, prefix=0, sms=SMS):
    up = lambda n: -(-n // 256) * 256  # noqa: E731
    group = q_heads // kv_heads
    rows = 128 // group * group
    tiles = -(-q_tokens * group // (2 * rows))
    base, pairs = tiles * kv_heads, max(sms // 2, 1)
    few = (group <= 16 and q_tokens <= seqs and k_tokens >= 16 * seqs and k_tokens > 0 and
           (prefix == 0 or (d == 64 and k_tokens >= 4096) or (d == 128 and k_tokens >= 32768)))
    keys = prefix + (0 if few else k_tokens)
    parts = max(min(pairs // base if base > 0 and base * 2 <= pairs else 1, -(-keys // 512)), 1)
    items = base * parts
    warps = -(-sms * 8 // kv_heads)
    chunk = max(-(-k_tokens // (warps - seqs if warps >= 8 * seqs else 5 * warps)), 64)
    chunk = -(-chunk // 16) * 16
    units = -(-k_tokens // chunk) + seqs if few else 0
    prow = parts * kv_heads * tiles * 2 * rows if parts > 1 or (few and prefix > 0) else 0
    frow = units * kv_heads * 16
    few_ml = up(up(256 + prow * 8) + prow * d * 4)
    size = 16 if prow == 0 and frow == 0 and items <= min(items, pairs) else up(few_ml + frow * 8) + frow * d * 4
    return Plan(few, parts, 1 if few and units // seqs + (parts if prefix else 0) <= 32 else 8, size)
