"""What is measured of the 4-bit paged KV cache: page allocation, the quantising append with its read-back,
and the attention over the cache. Each case runs either in a plain form (elementary torch operations)
or through the library's public calls, on the same inputs.

The cache of one layer is three tensors: the k codes and the v codes, two 4-bit codes a byte (element 2i in
the low half), [pages, page_size, heads, head_dim / 2] (NHD) or [pages, heads, page_size, head_dim / 2]
(HND), and bf16 [pages, heads, page_size, 4] holding (k scale, k minimum, v scale, v minimum) of each row. A row's
value is code * scale + minimum.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_TINY = 2.0 ** -126  # the least scale a row is stored with


# ---------------------------------------------------------------------------------------------------
# The cases.
# ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # One user's chat, a few hundred tokens in: the smallest call, where latency counts.
        dict(name="attend_one", kind="attend", batch=1, kv_min=517, kv_max=517, q_min=1, q_max=1, q_heads=32,
             kv_heads=8, head_dim=128, page_size=16, layout="NHD", dtype="bf16", lens_seed=0),
        # The decode rows of a mixed step at the 123B-class shape, ragged context lengths.
        dict(name="attend_decode", kind="attend", batch=256, kv_min=1, kv_max=4096, q_min=1, q_max=1, q_heads=96,
             kv_heads=8, head_dim=128, page_size=16, layout="NHD", dtype="bf16", lens_seed=1),
        # Few requests with long contexts (whole repositories in the prompt): the work has to be split along them.
        dict(name="attend_long", kind="attend", batch=8, kv_min=40000, kv_max=131072, q_min=1, q_max=1, q_heads=96,
             kv_heads=8, head_dim=128, page_size=16, layout="NHD", dtype="bf16", lens_seed=2),
        # Drafted tokens verified a few at a time, fp16, head-major pages.
        dict(name="attend_drafts", kind="attend", batch=48, kv_min=500, kv_max=8192, q_min=2, q_max=8, q_heads=32,
             kv_heads=8, head_dim=128, page_size=64, layout="HND", dtype="fp16", lens_seed=3),
        # Prompt chunks after a cached prefix, as a chunked prefill step runs them.
        dict(name="attend_prompt", kind="attend", batch=2, kv_min=5000, kv_max=8192, q_min=700, q_max=2048, q_heads=96,
             kv_heads=8, head_dim=128, page_size=16, layout="NHD", dtype="bf16", lens_seed=4),
        # Heads of 64 without sharing, pages of an odd size.
        dict(name="attend_small_heads", kind="attend", batch=31, kv_min=1, kv_max=3001, q_min=1, q_max=1, q_heads=12,
             kv_heads=12, head_dim=64, page_size=5, layout="NHD", dtype="fp16", lens_seed=5),
        # One new token for each of 64 running requests: the append of a decode step, read back.
        dict(name="append_decode", kind="append", batch=64, kv_min=1, kv_max=4096, q_min=1, q_max=1, kv_heads=8,
             head_dim=128, page_size=16, layout="NHD", dtype="bf16", lens_seed=6),
        # 64 ragged prompts of up to 1024 tokens after cached prefixes: the append of a prefill step, read back.
        dict(name="append_prompt", kind="append", batch=64, kv_min=1100, kv_max=8192, q_min=1, q_max=1024, kv_heads=8,
             head_dim=128, page_size=16, layout="NHD", dtype="bf16", lens_seed=7),
        # Heads of 64 in fp16, head-major pages of an odd size.
        dict(name="append_small_heads", kind="append", batch=17, kv_min=300, kv_max=3001, q_min=1, q_max=300,
             kv_heads=12, head_dim=64, page_size=5, layout="HND", dtype="fp16", lens_seed=8),
        # Pages for one more token of each of 256 running requests, then the step taken back.
        dict(name="pages_decode", kind="pages", batch=256, kv_min=1, kv_max=8192, q_min=1, q_max=1, page_size=16,
             lens_seed=9),
        # Pages for 64 ragged prompts, then the step taken back.
        dict(name="pages_prompt", kind="pages", batch=64, kv_min=1100, kv_max=8192, q_min=1, q_max=1024, page_size=16,
             lens_seed=10),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "pages"])
    page_size = rng.choice([1, 5, 16, 16, 16, 24, 32, 64])
    case = dict(kind=kind, page_size=page_size, lens_seed=rng.randrange(1 << 30))
    if kind == "pages":
        case["batch"] = _log_int(rng, 1, 1024)
        case["kv_max"] = _log_int(rng, 64, 8192)
        case["q_max"] = _log_int(rng, 1, min(case["kv_max"], 1 + 32768 // case["batch"]))
        case.update(kv_min=case["q_max"], q_min=rng.choice([0, 1]))
        return case
    head_dim = rng.choice([64, 128, 128])
    case.update(head_dim=head_dim, layout=rng.choice(["NHD", "HND"]), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "append":
        case["kv_heads"] = rng.choice([1, 2, 4, 5, 8, 12, 16])
        case["batch"] = _log_int(rng, 1, 256)
        case["kv_max"] = _log_int(rng, 16, 8192)
        budget = 65536 // case["kv_heads"] * 4 // case["batch"]
        case["q_max"] = _log_int(rng, 1, max(1, min(case["kv_max"], budget)))
        case.update(kv_min=case["q_max"], q_min=1)
        return case
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    case.update(kv_heads=kv_heads, q_heads=kv_heads * rng.choice([1, 2, 3, 4, 6, 8, 12, 12, 16]))
    form = rng.choice(["decode", "decode", "drafts", "prompt"])
    case["batch"] = _log_int(rng, 1, {"decode": 256, "drafts": 64, "prompt": 4}[form])
    limit = 131072 if form == "decode" else 8192
    tokens = {"decode": 4_500_000, "drafts": 2_000_000, "prompt": 65536}[form] // kv_heads
    case["kv_max"] = _log_int(rng, 16, max(16, min(limit, tokens // case["batch"])))
    q_max = {"decode": 1, "drafts": 8, "prompt": 1024}[form]
    case["q_max"] = 1 if form == "decode" else _log_int(rng, 2, max(2, min(q_max, case["kv_max"])))
    case["q_min"] = max(1, case["q_max"] // 2)
    case["kv_min"] = max(case["q_max"], case["kv_max"] // rng.choice([1, 2, 16]))
    return case


def _lengths(case):
    """(cached + new, new) tokens of each request: part of the case, whatever the seed of the values."""
    rng = random.Random(case["lens_seed"])
    kv = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(case["batch"])]
    new = [min(n, rng.randint(case["q_min"], case["q_max"])) for n in kv]
    return kv, new


def _blocks(n, page_size):
    return -(-n // page_size)


def work(case):
    kv, new = _lengths(case)
    tokens, ps = sum(new), case["page_size"]
    if case["kind"] == "pages":
        pages = sum(_blocks(n, ps) - _blocks(n - q, ps) for n, q in zip(kv, new))
        # allocate: both lengths in, seq_lens / last page / cumulative lengths out, batch index and position a
        # token, a free page read and a table entry written a page; release: lengths in and out, a page back.
        return {"bytes": case["batch"] * (8 + 12 + 8 + 4) + tokens * 8 + pages * (8 + 8), "flops": 0}
    d, h = case["head_dim"], case["kv_heads"]
    if case["kind"] == "append":
        # append: k and v in, codes and scales out; read: the same back. Index arithmetic beside it.
        return {"bytes": 2 * tokens * h * (4 * d + d + 8) + tokens * 16, "flops": tokens * h * 2 * d * 8}
    hq = case["q_heads"]
    seen = sum(q * (n - q) + q * (q + 1) // 2 for n, q in zip(kv, new))
    return {"bytes": sum(kv) * h * (d + 8) + 4 * tokens * hq * d + 4 * sum(_blocks(n, ps) for n in kv),
            "flops": 4 * d * hq * seen}


# ---------------------------------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------------------------------
def _tables(kv, page_size, gen, spare):
    """Block tables over a shuffled pool with `spare` unused pages; unused entries name the last page."""
    blocks = [_blocks(n, page_size) for n in kv]
    width = max(1, max(blocks))
    pool = sum(blocks) + spare
    perm = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(kv), width), pool - 1, dtype=torch.int32, device="cuda")
    count = torch.tensor(blocks, device="cuda")
    here = torch.arange(width, device="cuda")[None, :] < count[:, None]
    table[here] = perm[:sum(blocks)]
    return table, perm[sum(blocks):].contiguous(), pool


def _fill_cache(pool, heads, page_size, head_dim, layout, gen):
    """A cache in use: keys with strong channels, values without, quantised row by row."""
    shape = (pool, page_size, heads) if layout == "NHD" else (pool, heads, page_size)
    codes = [torch.empty(shape + (head_dim // 2,), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = torch.empty((pool, heads, page_size, 4), dtype=torch.bfloat16, device="cuda")
    channel = 1 + 3 * (torch.rand(head_dim, generator=gen, device="cuda") < 0.06).float()
    step = max(1, (1 << 24) // (heads * page_size * head_dim))
    for a in range(0, pool, step):
        n = min(step, pool - a)
        for which in range(2):
            x = torch.randn((n,) + shape[1:] + (head_dim,), generator=gen, device="cuda")
            x = x * channel if which == 0 else x
            low = x.amin(-1).to(torch.bfloat16)
            scale = ((x.amax(-1) - low.float()) / 15).to(torch.bfloat16)
            c = ((x - low.float()[..., None]) / scale.float()[..., None]).round().clamp(0, 15).to(torch.uint8)
            codes[which][a:a + n] = c[..., 0::2] | (c[..., 1::2] << 4)
            pair = torch.stack([scale, low], -1)
            scales[a:a + n, :, :, 2 * which:2 * which + 2] = pair.transpose(1, 2) if layout == "NHD" else pair
    return codes[0], codes[1], scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kv, new = _lengths(case)
    ps, batch = case["page_size"], case["batch"]
    state = dict(case=case, kv=kv, new=new)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["kind"] == "pages":
        # The pool holds what the requests have, what they are about to take, and some pages more.
        old = [n - q for n, q in zip(kv, new)]
        spare = sum(_blocks(n, ps) for n in kv) - sum(_blocks(n, ps) for n in old) + 7
        table, free, pool = _tables(old, ps, gen, spare)
        wide = torch.full((batch, max(1, _blocks(case["kv_max"], ps))), pool - 1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        state.update(append_lens=ints(new), seq_lens=ints(old), keep_lens=ints(old), block_tables=wide,
                     free_pages=free, num_free=ints([free.numel()]), tokens=sum(new))
        return state
    table, _, pool = _tables(kv, ps, gen, 3)
    dtype = _DTYPES[case["dtype"]]
    h, d = case["kv_heads"], case["head_dim"]
    tokens = sum(new)
    state.update(block_tables=table, seq_lens=ints(kv))
    if case["kind"] == "append":
        shape = (pool, ps, h, d // 2) if case["layout"] == "NHD" else (pool, h, ps, d // 2)
        state["cache"] = (torch.zeros(shape, dtype=torch.uint8, device="cuda"),
                          torch.zeros(shape, dtype=torch.uint8, device="cuda"),
                          torch.zeros((pool, h, ps, 4), dtype=torch.bfloat16, device="cuda"))
        channel = 1 + 3 * (torch.rand(d, generator=gen, device="cuda") < 0.06).float()
        # k and v are column ranges of one row, as the fused projection writes them.
        rows = torch.randn((tokens, 2, h, d), generator=gen, device="cuda")
        rows[:, 0] *= channel
        rows = rows.to(dtype)
        lens = ints(new)
        state.update(
            key=rows[:, 0], value=rows[:, 1],
            batch_indices=torch.repeat_interleave(torch.arange(batch, dtype=torch.int32, device="cuda"), lens,
                                                  output_size=tokens),
            positions=ints([p for n, q in zip(kv, new) for p in range(n - q, n)]),
            kv_indptr=torch.arange(batch + 1, dtype=torch.int32, device="cuda") * table.shape[1],
            kv_last_page_len=ints([(n - 1) % ps + 1 if n else 0 for n in kv]))
        return state
    state["cache"] = _fill_cache(pool, h, ps, d, case["layout"], gen)
    # Rotated queries: near unit scale, some heads sharper than others.
    sharp = 0.5 + 1.5 * torch.rand((1, case["q_heads"], 1), generator=gen, device="cuda")
    state["query"] = (torch.randn((tokens, case["q_heads"], d), generator=gen, device="cuda") * sharp).to(dtype)
    starts = [0]
    for q in new:
        starts.append(starts[-1] + q)
    state.update(starts=starts, cum_q=ints(starts))
    return state


# ---------------------------------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": _attend_own, "append": _append_own, "pages": _pages_own}[kind](state)
    return {"attend": _attend_plain, "append": _append_plain, "pages": _pages_plain}[kind](state)


def _attend_own(s):
    import mas_b200

    decode = s["case"]["q_max"] == 1
    return mas_b200.paged_attention_int4(s["query"], s["cache"], s["block_tables"], s["seq_lens"],
                                         cum_seq_lens_q=None if decode else s["cum_q"], kv_layout=s["case"]["layout"])


def _append_own(s):
    import mas_b200

    layout = s["case"]["layout"]
    indices = s["block_tables"].flatten()
    mas_b200.append_paged_kv_cache_int4(s["key"], s["value"], s["batch_indices"], s["positions"], s["cache"], indices,
                                        s["kv_indptr"], s["kv_last_page_len"], kv_layout=layout)
    return mas_b200.read_paged_kv_cache_int4(s["batch_indices"], s["positions"], s["cache"], indices, s["kv_indptr"],
                                             dtype=s["key"].dtype, kv_layout=layout)


def _pages_own(s):
    import mas_b200

    ps = s["case"]["page_size"]
    maps = mas_b200.allocate_paged_kv(s["append_lens"], s["seq_lens"], s["block_tables"], s["free_pages"],
                                      s["num_free"], ps, s["tokens"])
    mas_b200.release_paged_kv(s["keep_lens"], s["seq_lens"], s["block_tables"], s["free_pages"], s["num_free"], ps)
    return (*maps, s["block_tables"], s["seq_lens"], s["free_pages"], s["num_free"])


def _rows_of(cache, layout, pages, entries):
    """Codes as fp32 [2, tokens, heads, head_dim] and scales [tokens, heads, 4] of the named cache rows."""
    out = []
    for codes in cache[:2]:
        c = codes[pages, entries] if layout == "NHD" else codes[pages, :, entries]
        out.append(torch.stack([c & 15, c >> 4], -1).flatten(-2).float())
    return out, cache[2][pages, :, entries].float()


def _attend_plain(s):
    case = s["case"]
    ps, h, d, hq = case["page_size"], case["kv_heads"], case["head_dim"], case["q_heads"]
    out = torch.empty_like(s["query"])
    for b, n in enumerate(s["kv"]):
        if n == 0:
            out[s["starts"][b]:s["starts"][b + 1]] = 0
            continue
        t = torch.arange(n, device="cuda")
        (k, v), sc = _rows_of(s["cache"], case["layout"], s["block_tables"][b].long()[t // ps], t % ps)
        q = s["query"][s["starts"][b]:s["starts"][b + 1]].float()
        m = q.shape[0]
        hidden = t[None, :] > (n - m + torch.arange(m, device="cuda"))[:, None]
        for j in range(h):
            kj = k[:, j] * sc[:, j, 0:1] + sc[:, j, 1:2]
            vj = v[:, j] * sc[:, j, 2:3] + sc[:, j, 3:4]
            qj = q[:, j * (hq // h):(j + 1) * (hq // h)]
            x = torch.einsum("mgd,td->gmt", qj, kj) * (1 / math.sqrt(d))
            x.masked_fill_(hidden, float("-inf"))
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.einsum("gmt,td->mgd", x, vj) / x.sum(-1).t()[..., None]
            out[s["starts"][b]:s["starts"][b + 1], j * (hq // h):(j + 1) * (hq // h)] = o.to(out.dtype)
    return out


def _down_bf16(x):
    """The largest bf16 not above each fp32 value."""
    y = x.to(torch.bfloat16).float()
    low = torch.nextafter(y.to(torch.bfloat16), torch.full_like(y, float("-inf"), dtype=torch.bfloat16)).float()
    return torch.where(y > x, low, y)


def _quantise_plain(x):
    """Codes, scale and minimum of rows, the steps near a border in 64 bits."""
    low = _down_bf16(x.amin(-1).float()).double()
    y = (x.amax(-1).double() - low) / 15
    scale = (-_down_bf16((-y).float())).double()
    # (-y) in fp32 may have been rounded away from the border: put the scale back to the least that covers the row
    top = x.amax(-1).double() - low
    up = torch.nextafter(scale.to(torch.bfloat16), torch.full_like(scale, float("inf"), dtype=torch.bfloat16)).double()
    down = torch.nextafter(scale.to(torch.bfloat16), torch.full_like(scale, float("-inf"),
                                                                      dtype=torch.bfloat16)).double()
    scale = torch.where(15 * scale < top, up, torch.where(15 * down >= top, down, scale)).clamp(min=_TINY)
    diff = (x.double() - low[..., None]).float().double()
    return torch.floor(diff / scale[..., None] + 0.5).to(torch.uint8), scale.float(), low.float()


def _append_plain(s):
    case = s["case"]
    ps, layout = case["page_size"], case["layout"]
    pos = s["positions"].long()
    pages = s["block_tables"].flatten().long()[s["kv_indptr"].long()[s["batch_indices"].long()] + pos // ps]
    entries = pos % ps
    for which, x in enumerate((s["key"], s["value"])):
        c, scale, low = _quantise_plain(x)
        packed = c[..., 0::2] | (c[..., 1::2] << 4)
        if layout == "NHD":
            s["cache"][which][pages, entries] = packed
        else:
            s["cache"][which][pages, :, entries] = packed
        s["cache"][2][pages, :, entries, 2 * which] = scale.to(torch.bfloat16)
        s["cache"][2][pages, :, entries, 2 * which + 1] = low.to(torch.bfloat16)
    (k, v), sc = _rows_of(s["cache"], layout, pages, entries)
    return ((k * sc[..., 0:1] + sc[..., 1:2]).to(s["key"].dtype), (v * sc[..., 2:3] + sc[..., 3:4]).to(s["key"].dtype))


def _pages_plain(s):
    ps = s["case"]["page_size"]
    app, lens, table, free, num = (s["append_lens"], s["seq_lens"], s["block_tables"], s["free_pages"], s["num_free"])
    total = lens + app
    have, want = (lens + ps - 1) // ps, (total + ps - 1) // ps
    cum = torch.cat([torch.zeros_like(num), app.cumsum(0)]).to(torch.int32)
    token = torch.arange(s["tokens"], dtype=torch.int32, device="cuda")
    batch = torch.searchsorted(cum[1:], token, right=True).to(torch.int32)
    positions = token - cum[batch.long()] + lens[batch.long()]
    last = torch.where(total > 0, (total - 1) % ps + 1, 0).to(torch.int32)
    need = want - have
    before = need.cumsum(0) - need
    column = torch.arange(table.shape[1], device="cuda")[None, :]
    rank = before[:, None] + column - have[:, None]
    fresh = (column >= have[:, None]) & (column < want[:, None])
    source = (num - 1 - rank).clamp(0, free.numel() - 1).long()
    table.copy_(torch.where(fresh, free[source], table))
    num -= need.sum().to(torch.int32)
    lens.copy_(total)
    # the step taken back: pages past the kept lengths return so that the next pop finds them in the same order
    keep = (s["keep_lens"] + ps - 1) // ps
    back = want - keep
    all_back = back.sum()
    rank = (back.cumsum(0) - back)[:, None] + column - keep[:, None]
    gone = (column >= keep[:, None]) & (column < want[:, None])
    slot = torch.where(gone, num + all_back - 1 - rank, free.numel()).long()
    grown = torch.cat([free, free[:1]])
    grown.scatter_(0, slot.flatten(), table.flatten())
    free.copy_(grown[:-1])
    num += all_back.to(torch.int32)
    lens.copy_(s["keep_lens"])
    return cum, batch, positions, last, table, lens, free, num


# ---------------------------------------------------------------------------------------------------
# From the definitions, in 64 bits.
# ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    ps = case["page_size"]
    if case["kind"] == "pages":
        return None  # whole numbers only
    if case["kind"] == "append":
        result = []
        for x in (s["key"], s["value"]):
            x64 = x.double()
            low, high = x64.min(-1, keepdim=True).values, x64.max(-1, keepdim=True).values
            one = torch.ones_like(low)
            unit = torch.ldexp(one, torch.frexp(low.abs().clamp(min=_TINY)).exponent - 8)  # a bf16 step at |low|
            low = torch.floor(low / unit) * unit
            need = high - low
            guess = (need / 15).clamp(min=_TINY)
            unit = torch.ldexp(one, torch.frexp(guess).exponent - 8)
            steps = torch.floor(guess / unit) - 1
            for _ in range(3):
                steps = torch.where(steps * unit * 15 < need, steps + 1, steps)
            scale = (steps * unit).clamp(min=_TINY)
            code = torch.floor((x64 - low).float().double() / scale + 0.5).clamp(0, 15)
            result.append(code * scale + low)
        return tuple(result)
    q, (ck, cv, scales) = s["query"].double(), s["cache"]
    h, group, d = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"]
    if case["layout"] == "HND":
        ck, cv = ck.transpose(1, 2), cv.transpose(1, 2)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["kv"]):
        pages = s["block_tables"][b, :_blocks(n, ps)].long()
        first, m = s["starts"][b], s["new"][b]
        order = torch.arange(n, device="cuda")
        for j in range(h):
            pair = scales[pages, j].double().reshape(-1, 4)[:n]
            mats = []
            for i, c in enumerate((ck, cv)):
                byte = c[pages, :, j].reshape(-1, d // 2)[:n]
                val = torch.empty((n, d), dtype=torch.float64, device="cuda")
                val[:, 0::2] = (byte % 16).double()
                val[:, 1::2] = (byte // 16).double()
                mats.append(val * pair[:, 2 * i, None] + pair[:, 2 * i + 1, None])
            rows = q[first:first + m, j * group:(j + 1) * group].reshape(m * group, d)
            logits = rows @ mats[0].t() / math.sqrt(d)
            limit = n - m + torch.arange(m, device="cuda").repeat_interleave(group)
            logits = logits.masked_fill(order[None, :] > limit[:, None], float("-inf"))
            out[first:first + m, j * group:(j + 1) * group] = (torch.softmax(logits, -1) @ mats[1]).view(m, group, d)
    return out
