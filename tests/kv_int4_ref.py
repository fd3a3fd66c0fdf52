"""Plain 64-bit forms of the 4-bit paged cache's operators, on the CPU, for the tests.

Written from the definitions: the row format (minimum m = the largest bf16 <= min x, scale s = the least bf16
>= max(2^-126, (max x - m) / 15), code floor(f32(x - m) / s + 1/2), value c s + m), the stack of free pages, and
softmax(sm_scale q k^T) v. Sums over a row's exact fractions use Python's Fraction where a border decides.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch


def bf16_steps(value: Fraction, up: bool) -> float:
    """The nearest bf16 at or above (up) / at or below a finite rational, as a float."""
    x = torch.tensor(float(value), dtype=torch.float64)
    y = x.to(torch.bfloat16)
    while Fraction(y.item()) < value if up else Fraction(y.item()) > value:
        y = torch.nextafter(y, torch.full_like(y, math.inf if up else -math.inf))
    while True:
        z = torch.nextafter(y, torch.full_like(y, -math.inf if up else math.inf))
        if Fraction(z.item()) < value if up else Fraction(z.item()) > value:
            return y.item()
        y = z


def quantise_row(x: torch.Tensor) -> tuple[list[int], float, float]:
    """(codes, scale, minimum) of one row, by exact rational arithmetic."""
    vals = x.double().tolist()
    if not all(math.isfinite(v) for v in vals):
        return [0] * len(vals), math.nan, math.nan
    low = bf16_steps(Fraction(min(vals)), up=False)
    scale = bf16_steps(max((Fraction(max(vals)) - Fraction(low)) / 15, Fraction(2) ** -126), up=True)
    codes = []
    for v in vals:
        # the difference rounds in fp32; halves keep it in range
        half = torch.tensor(v / 2 - low / 2, dtype=torch.float64).to(torch.float32).item()
        codes.append(math.floor(2 * Fraction(half) / Fraction(scale) + Fraction(1, 2)))
    return codes, scale, low


def read_rows(cache, layout: str, pages, entries):
    """fp64 (k, v) [tokens, heads, D] of the named cache rows, and the codes behind them."""
    out = []
    pairs = cache[2].double()
    for which, codes in enumerate(cache[:2]):
        c = codes[pages, entries] if layout == "NHD" else codes[pages, :, entries]
        c = torch.stack([c & 15, c >> 4], -1).flatten(-2).double()
        pr = pairs[pages, :, entries]
        out.append(c * pr[..., 2 * which, None] + pr[..., 2 * which + 1, None])
    return out


def attention(q, cache, layout, tables, seq_lens, cum_q, sm_scale, causal=True):
    """(out fp64 [T, Hq, D], lse in log2 [T, Hq], covered [T]); rows no request covers stay NaN."""
    T, hq, d = q.shape
    page_size = cache[2].shape[2]
    h = cache[2].shape[1]
    out = torch.full((T, hq, d), math.nan, dtype=torch.float64)
    lse = torch.full((T, hq), math.nan, dtype=torch.float64)
    for b, n in enumerate(seq_lens):
        q0, q1 = cum_q[b], cum_q[b + 1]
        tok = torch.arange(n)
        k, v = read_rows(cache, layout, tables[b].long()[tok // page_size], tok % page_size)
        for i in range(q0, q1):
            seen = max(0, min(n, n - (q1 - q0) + (i - q0) + 1)) if causal else n
            if seen == 0:
                out[i], lse[i] = 0, -math.inf
                continue
            qi = q[i].double().view(h, hq // h, d)
            s = torch.einsum("hgd,thd->hgt", qi, k[:seen]) * sm_scale
            out[i] = torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), v[:seen]).reshape(hq, d)
            lse[i] = (torch.logsumexp(s, -1) / math.log(2)).reshape(hq)
    return out, lse


def allocate(append, seq_lens, table, free, num_free, page_size, max_tokens):
    """Python lists in, (ok, cum, batch, pos, last, seq_lens, table, num_free) out; the inputs stay."""
    pages = lambda n: -(-n // page_size)  # noqa: E731
    width = len(table[0]) if table else 0
    ok = all(a >= 0 and n >= 0 and n + a <= width * page_size for a, n in zip(append, seq_lens))
    need = [pages(n + a) - pages(n) for a, n in zip(append, seq_lens)]
    ok = ok and 0 <= num_free <= len(free) and sum(need) <= num_free and sum(append) <= max_tokens
    last = lambda n: (n - 1) % page_size + 1 if n > 0 else 0  # noqa: E731
    if not ok:
        return (False, [0] * (len(append) + 1), [-1] * max_tokens, [0] * max_tokens, [last(n) for n in seq_lens],
                list(seq_lens), [list(r) for r in table], num_free)
    table = [list(r) for r in table]
    cum, batch, pos = [0], [], []
    for b, (a, n) in enumerate(zip(append, seq_lens)):
        for j in range(pages(n), pages(n + a)):
            num_free -= 1
            table[b][j] = free[num_free]
        batch += [b] * a
        pos += range(n, n + a)
        cum.append(cum[-1] + a)
    pad = max_tokens - len(batch)
    new = [n + a for a, n in zip(append, seq_lens)]
    return True, cum, batch + [-1] * pad, pos + [0] * pad, [last(n) for n in new], new, table, num_free


def release(keep, seq_lens, table, free, num_free, page_size):
    """(ok, seq_lens, free, num_free)."""
    pages = lambda n: -(-n // page_size)  # noqa: E731
    back = [table[b][j] for b, (k, n) in enumerate(zip(keep, seq_lens)) if 0 <= k <= n
            for j in range(pages(k), pages(n))]
    if not all(0 <= k <= n for k, n in zip(keep, seq_lens)) or not 0 <= num_free <= len(free) - len(back):
        return False, list(seq_lens), list(free), num_free
    free = list(free)
    for p in reversed(back):
        free[num_free] = p
        num_free += 1
    return True, list(keep), free, num_free
