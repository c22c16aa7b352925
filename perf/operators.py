"""The operators of serving in 8 bits: block tables, the paged K/V cache, its attention, the 8-bit product.

One step of a server that holds its K/V in 8 bits runs them in this order: ``plan`` turns the number
of new tokens of every request into block tables and slot maps; ``linear`` makes q, k and v (rows
quantised to e4m3 with a scale for each 128 values, times weights held in e4m3 with a scale for each
128 x 128 block); ``append`` puts k and v into the cache (blocks of 64 tokens, one scale for each block
and head; a request's last, unfilled block stays in 16 bits); ``attend`` reads it.

``run`` computes them in elementary torch operations, or, where ``own`` is true, through the package's
public calls on the same tensors. ``exact`` evaluates the same definitions in float64.
"""
import math
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "tsfm-zig_amd"))

own = False

BLOCK = 64  # tokens of a cache block
GROUP = 128  # values (and weight rows) that share a scale of the 8-bit product
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}


# ---- the cases --------------------------------------------------------------------------------------


def listed():
    return [
        # A decode step's bookkeeping: one token for each of 256 running requests. Launches and latency.
        dict(name="plan_decode", kind="plan", requests=256, max_len=8192, new=1),
        # Admission of 1024 prompts of 0 to 512 tokens on top of cached prefixes.
        dict(name="plan_prompts", kind="plan", requests=1024, max_len=2048, new=512),
        # The K/V of one decode step into the cache: 256 requests, 16 heads, most tokens go to a tail.
        dict(name="append_decode", kind="append", requests=256, max_len=128, new=1, kv_heads=16, head_dim=64,
             code="e4m3", dtype="bf16"),
        # The K/V of 16 prompts of up to 2048 tokens, grouped heads.
        dict(name="append_prompts", kind="append", requests=16, max_len=0, new=2048, kv_heads=8, head_dim=128,
             code="i8", dtype="f16"),
        # One interactive request: a token over 300 cached ones. Latency.
        dict(name="attend_one", kind="attend", requests=1, max_len=300, new=1, heads=16, kv_heads=16, head_dim=64,
             code="e4m3", dtype="bf16"),
        # A decode step of 128 requests of 1 to 4096 tokens.
        dict(name="attend_batch", kind="attend", requests=128, max_len=4096, new=1, heads=16, kv_heads=16, head_dim=64,
             code="e4m3", dtype="bf16"),
        # Two requests with very long contexts, grouped heads: few rows, the work is one long axis.
        dict(name="attend_long", kind="attend", requests=2, max_len=262144, new=1, heads=32, kv_heads=8, head_dim=128,
             code="i8", dtype="f16"),
        # Decode blocks of 32 tokens (32 forecast patches at a time), 64 requests of up to 1024 tokens.
        dict(name="attend_blocks", kind="attend", requests=64, max_len=1024, new=32, heads=16, kv_heads=16, head_dim=64,
             code="e4m3", dtype="bf16"),
        # Prompts in chunks of up to 2048 tokens over up to 8192 cached ones: compute bound.
        dict(name="attend_prompts", kind="attend", requests=4, max_len=8192, new=2048, heads=32, kv_heads=8,
             head_dim=128, code="e4m3", dtype="bf16"),
        # The product of a single token's row, f32 in and out as the framework's f32 families have it.
        dict(name="linear_one", kind="linear", m=1, n=1024, k=1024, dtype="f32", out="f32"),
        # A ragged batch of 2331 tokens through a layer's up projection.
        dict(name="linear_ragged", kind="linear", m=2331, n=4096, k=1024, dtype="bf16", out="bf16"),
        # A large batch through a wide layer.
        dict(name="linear_large", kind="linear", m=16384, n=8192, k=4096, dtype="bf16", out="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "linear", "linear"])
    if kind == "plan":
        return dict(kind=kind, requests=_log_int(rng, 1, 1024), max_len=_log_int(rng, 64, 8192),
                    new=rng.choice([1, _log_int(rng, 2, 512)]))
    heads, kv_heads = rng.choice([(16, 16), (12, 12), (32, 8), (8, 1), (24, 8), (7, 7)])
    half = dict(head_dim=rng.choice([64, 128]), code=rng.choice(["e4m3", "i8"]), dtype=rng.choice(["bf16", "f16"]))
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, requests=_log_int(rng, 1, 256), max_len=_log_int(rng, 2, 128), new=1,
                        kv_heads=kv_heads, **half)
        return dict(kind=kind, requests=_log_int(rng, 1, 16), max_len=0, new=_log_int(rng, 2, 2048),
                    kv_heads=kv_heads, **half)
    if kind == "attend":
        new = rng.choice([1, 1, 32, _log_int(rng, 2, 1024)])
        max_len = max(new + 1, _log_int(rng, 32, 32768))
        # as much work as the listed cases at most: keys read, and pairs scored
        most = min(128, 2 * 262144 * 8 * 128 // (max_len * kv_heads * half["head_dim"]),
                   4 * 2048 * 8192 * 32 * 128 // (2 * new * max_len * heads * half["head_dim"]))
        return dict(kind=kind, requests=_log_int(rng, 1, max(1, most)), max_len=max_len, new=new, heads=heads,
                    kv_heads=kv_heads, **half)
    return dict(kind=kind, m=_log_int(rng, 1, 8192), n=_log_int(rng, 64, 8192), k=16 * _log_int(rng, 16, 256),
                dtype=rng.choice(["f32", "bf16", "f16"]), out=rng.choice(["f32", "bf16", "f16"]))


def _spread(case):
    """(tokens held before the pass, new tokens) of every request: the same for every seed but for their order.
    Lengths are spread evenly; of several new tokens some requests have none, most have fewer than the most."""
    r, new, top = case["requests"], case["new"], case["max_len"]
    held = [(i + 1) * top // r for i in range(r)]
    fresh = [new if new in (1, 32) else (new * ((7 * i) % r + 1)) // r for i in range(r)]
    if case["kind"] == "append" or (new > 1 and r > 3 and case["kind"] == "plan"):
        fresh = [0 if r > 3 and new > 1 and i % 8 == 5 else n for i, n in enumerate(fresh)]
    fresh[-1] = new
    if case["kind"] == "attend":  # max_len counts the new tokens, as attention reads them
        held = [max(0, h - n) for h, n in zip(held, fresh)]
    return held, fresh


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        size = {"f32": 4, "bf16": 2, "f16": 2}
        kb = _blocks_of(k)
        return {"bytes": m * k * size[case["dtype"]] + m * k + 4 * m * kb + n * k + 4 * _blocks_of(n) * kb
                + m * n * size[case["out"]], "flops": 2 * m * n * k}
    held, fresh = _spread(case)
    r, tokens = len(held), sum(fresh)
    if case["kind"] == "plan":
        taken = sum(_blocks(h + n) - _blocks(h) for h, n in zip(held, fresh))
        items = sum((h + n - 1) // BLOCK - h // BLOCK + 1 for h, n in zip(held, fresh) if n)
        return {"bytes": r * 4 * 6 + taken * 8 + tokens * 12 + items * 8 + 24, "flops": tokens + 4 * r}
    kv, d = case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        full = sum((h + n) // BLOCK - h // BLOCK for h, n in zip(held, fresh))
        old = sum(h % BLOCK for h, n in zip(held, fresh) if (h + n) // BLOCK > h // BLOCK)
        tail = sum((h + n) - max(h, (h + n) // BLOCK * BLOCK) for h, n in zip(held, fresh))
        row = 2 * kv * d
        return {"bytes": (tokens + old + tail) * row * 2 + full * (BLOCK * row + 8 * kv), "flops": 3 * tokens * row}
    total = [h + n for h, n in zip(held, fresh)]
    keys = sum(t for t, n in zip(total, fresh) if n)
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, fresh))
    return {"bytes": keys * kv * d * 2 + tokens * case["heads"] * d * 4, "flops": 4 * pairs * case["heads"] * d}


def _blocks_of(n):
    return -(-n // GROUP)


# ---- inputs -----------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype=torch.float32, step=1 << 26):
    """Normal values, made in pieces (the cache of a long context is larger than one f32 copy should be)."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), step):
        piece = flat[at:at + step]
        piece.copy_(torch.randn(piece.numel(), generator=g, device="cuda"))
    return out


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _lengths(case, seed):
    """held and fresh tokens of the requests, in the seed's order."""
    held, fresh = _spread(case)
    order = torch.randperm(len(held), generator=torch.Generator().manual_seed(int(seed))).tolist()
    return [held[i] for i in order], [fresh[i] for i in order]


def _pick(x, *at):
    """x[at] of a tensor of 8-bit values (indexed as bytes: not every torch operation knows the type)."""
    return x.view(torch.int8)[at].view(x.dtype)


def _prefix(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _items_room(requests, tokens):
    return min(tokens, tokens // BLOCK + 2 * requests)


def _table(g, counts, width, blocks):
    """Block tables: a random order of the pool's blocks, dealt to the requests; -1 where a row has none."""
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    start = torch.tensor(_prefix(counts)[:-1], device="cuda")
    j = torch.arange(width, device="cuda")
    at = start[:, None] + j[None]
    have = j[None] < torch.tensor(counts, device="cuda")[:, None]
    return torch.where(have, order[at.clamp(max=blocks - 1)], torch.full_like(order[:1], -1)), order


def _prepare_plan(case, seed):
    g = _gen(seed)
    held, fresh = _lengths(case, seed)
    r, tokens = len(held), sum(fresh)
    width = _blocks(max(h + n for h, n in zip(held, fresh))) + 1
    counts = [_blocks(h) for h in held]
    used = sum(counts)
    blocks = used + sum(_blocks(h + n) - c for h, n, c in zip(held, fresh, counts)) + 7
    table, order = _table(g, counts, width, blocks)
    free = torch.full((blocks,), -1, dtype=torch.int32, device="cuda")
    free[:blocks - used] = order[used:]
    room, items = tokens + 5, _items_room(r, tokens + 5)  # a server's arrays are a little longer than one step's tokens
    return dict(kind="plan", blocks=blocks, n_new=_i32(fresh), length=_i32(held), free_list=free,
                free_count=_i32([blocks - used]), table=table, length_out=torch.empty_like(_i32(held)),
                free_count_out=_i32([0]), cu_tokens=torch.empty(r + 1, dtype=torch.int32, device="cuda"),
                cu_blocks=torch.empty(r + 1, dtype=torch.int32, device="cuda"),
                cu_items=torch.empty(r + 1, dtype=torch.int32, device="cuda"),
                slots=torch.empty(room, dtype=torch.int64, device="cuda"),
                pos=torch.empty(room, dtype=torch.int32, device="cuda"),
                items=torch.empty((items, 2), dtype=torch.int32, device="cuda"),
                status=torch.empty(4, dtype=torch.int32, device="cuda"))


def _cache(g, case, total, held):
    """A cache that holds the lengths `total`, the K/V of the first `held` tokens of each request in it: quantised
    blocks of normal values (keys with a few large channels, as projections have them), and tails."""
    kv, d, code, dtype = case["kv_heads"], case["head_dim"], CODES[case["code"]], DTYPES[case["dtype"]]
    counts = [_blocks(t) for t in total]
    blocks, width = sum(counts) + 1, max(1, max(counts))
    table, _ = _table(g, counts, width, blocks - 1)  # the last block belongs to no request
    r = len(total)
    c = dict(k=torch.zeros((blocks, kv, BLOCK, d), dtype=torch.int8, device="cuda").view(code),
             v=torch.zeros((blocks, kv, d, BLOCK), dtype=torch.int8, device="cuda").view(code),
             scales=torch.ones((blocks, kv, 2), device="cuda"), table=table, length=_i32(total),
             k_tail=_normal(g, (r, kv, BLOCK, d), dtype), v_tail=_normal(g, (r, kv, BLOCK, d), dtype))
    loud = torch.ones(d, device="cuda")
    loud[::17] = 4.0
    c["k_tail"] *= loud.to(dtype)
    if max(held):
        step = max(1, (1 << 26) // (kv * BLOCK * d))
        for at in range(0, blocks, step):
            n = min(step, blocks - at)
            for name, gain, which in (("k", loud, 0), ("v", 1.0, 1)):
                x = torch.randn((n, kv, BLOCK, d), generator=g, device="cuda") * gain
                codes, s = _quantise(x.to(dtype).float(), (2, 3), case["code"])
                c[name][at:at + n] = codes if name == "k" else _to_v(codes)
                c["scales"][at:at + n, :, which] = s
    return c


def _prepare_append(case, seed):
    g = _gen(seed)
    held, fresh = _lengths(case, seed)
    total = [h + n for h, n in zip(held, fresh)]
    tokens, row = sum(fresh), case["kv_heads"] * case["head_dim"]
    dtype = DTYPES[case["dtype"]]
    kv = _normal(g, (tokens, 2 * row), dtype)  # k and v as a fused projection leaves them
    items = [(i, j) for i, (h, n) in enumerate(zip(held, fresh)) if n for j in range(h // BLOCK, (h + n - 1) // BLOCK + 1)]
    room = _items_room(len(held), tokens)
    items += [(-1, -1)] * (room - len(items))
    s = dict(kind="append", code=case["code"], k_new=kv[:, :row], v_new=kv[:, row:], cu_tokens=_i32(_prefix(fresh)),
             items=_i32(items), **_cache(g, case, total, [0]))
    if own:
        import tsfm_attn

        s["cache"] = tsfm_attn.Kv8Cache(**{n: s[n] for n in ("k", "v", "scales", "k_tail", "v_tail", "table", "length")})
    return s


def _prepare_attend(case, seed):
    g = _gen(seed)
    held, fresh = _lengths(case, seed)
    total = [h + n for h, n in zip(held, fresh)]
    tokens, heads, d = sum(fresh), case["heads"], case["head_dim"]
    s = dict(kind="attend", code=case["code"], q=_normal(g, (tokens, heads, d), DTYPES[case["dtype"]]),
             cu_tokens=_i32(_prefix(fresh)), most_new=max(fresh), most_len=max(total), scale=1.0 / math.sqrt(d),
             **_cache(g, case, total, total))
    s["o"] = torch.empty_like(s["q"])
    if own:
        import tsfm_attn

        s["cache"] = tsfm_attn.Kv8Cache(**{n: s[n] for n in ("k", "v", "scales", "k_tail", "v_tail", "table", "length")})
        s["workspace"] = torch.empty(tsfm_attn.kv8_attend_workspace(
            s["cache"], heads=heads, tokens=tokens, max_new=s["most_new"], max_len=s["most_len"]),
            dtype=torch.uint8, device="cuda")
    return s


def _prepare_linear(case, seed):
    g = _gen(seed)
    m, n, k = case["m"], case["n"], case["k"]
    x = _normal(g, (m, k)) * torch.exp(torch.randn((m, 1), generator=g, device="cuda"))  # rows of different loudness
    w = _normal(g, (n, k)) * k ** -0.5
    pad = torch.zeros((_blocks_of(n) * GROUP, _blocks_of(k) * GROUP), device="cuda")
    pad[:n, :k] = w
    tiles = pad.view(_blocks_of(n), GROUP, _blocks_of(k), GROUP)
    # A checkpoint's weights: scales of any value, absmax / 448
    b_scales = (tiles.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp_min(2.0 ** -100)
    b = (tiles / b_scales[:, None, :, None]).to(torch.float8_e4m3fn).view_as(pad)[:n, :k].contiguous()
    return dict(kind="linear", x=x.to(DTYPES[case["dtype"]]), b=b, b_scales=b_scales.contiguous(),
                a=torch.empty((m, k), dtype=torch.float8_e4m3fn, device="cuda"),
                a_scales=torch.empty((m, _blocks_of(k)), device="cuda"),
                y=torch.empty((m, n), dtype=DTYPES[case["out"]], device="cuda"))


def prepare(case, seed):
    return {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend,
            "linear": _prepare_linear}[case["kind"]](case, seed)


# ---- plain forms ------------------------------------------------------------------------------------


def _power_of_two_scale(amax):
    """The smallest power of two s (2^-126 at least) with amax / s <= 448; 1 for a group of zeros."""
    frac, e = torch.frexp(amax)  # amax = frac 2^e, frac in [1/2, 1); 448 = 0.875 * 2^9
    e = (e.to(torch.int32) - 9 + (frac > 0.875).to(torch.int32)).clamp(min=-126)
    s = ((e + 127) << 23).view(torch.float32)  # from its bits: a power function need not be exact
    return torch.where(amax > 0, s, torch.ones_like(s))


def _quantise(x, dims, code):
    """f32 values -> (codes, scale of each group): a group is what `dims` spans."""
    amax = x.abs().amax(dim=dims, keepdim=True)
    if code == "e4m3":
        s = _power_of_two_scale(amax)
        return (x / s).to(torch.float8_e4m3fn), s.flatten(-len(dims)).squeeze(-1)
    top = amax.clamp_min(2.0 ** -100)
    s = torch.where(amax > 0, top / 127.0, torch.ones_like(amax))
    return torch.round(x * (127.0 / top)).clamp(-127, 127).to(torch.int8), s.flatten(-len(dims)).squeeze(-1)


# In a block of V, the 64 tokens of one dim lie in the order in which the matrix instructions take them: token
# 32 c + 16 a + 4 g + i at byte 16 g + 8 c + 4 a + i.
def _to_v(codes):
    """(..., 64 tokens, d) -> (..., d, 64 bytes)."""
    t = codes.view(torch.int8).transpose(-1, -2)
    t = t.unflatten(-1, (2, 2, 4, 4)).movedim(-2, -4)  # (c, a, g, i) -> (g, c, a, i)
    return t.reshape(*codes.shape[:-2], codes.shape[-1], BLOCK).view(codes.dtype)


def _from_v(v):
    """(..., d, 64 bytes) -> (..., 64 tokens, d), f32."""
    t = v.float().unflatten(-1, (4, 2, 2, 4)).movedim(-4, -2)  # (g, c, a, i) -> (c, a, g, i)
    return t.reshape(*v.shape[:-1], BLOCK).transpose(-1, -2)


def _plain_plan(s):
    length, n = s["length"].long(), s["n_new"].long()
    width, room = s["table"].shape[1], s["slots"].numel()
    dev = n.device
    total, taken = length + n, (length + n + BLOCK - 1) // BLOCK - (length + BLOCK - 1) // BLOCK
    short = taken.sum() > s["free_count"][0]
    code = torch.where(n.sum() > room, 1, torch.where((total > width * BLOCK).any(), 2, torch.where(short, 3, 0)))
    n, taken = torch.where(code == 0, n, 0), torch.where(code == 0, taken, 0)
    total = length + n
    zero = torch.zeros(1, dtype=torch.long, device=dev)
    cu, cb = torch.cat([zero, n.cumsum(0)]), torch.cat([zero, taken.cumsum(0)])
    # the new blocks of a request are the next ones from the end of the free list
    j = torch.arange(width, device=dev)[None]
    first = (length + BLOCK - 1) // BLOCK
    new = (j >= first[:, None]) & (j < (first + taken)[:, None])
    at = s["free_count"].long()[0] - 1 - cb[:-1, None] - (j - first[:, None])
    s["table"].copy_(torch.where(new, s["free_list"][at.clamp(0, s["blocks"] - 1)], s["table"]))
    t = torch.arange(room, device=dev)
    live = t < cu[-1]
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=n.numel() - 1)
    pos = length[r] + t - cu[r]
    block = s["table"][r, (pos // BLOCK).clamp(0, width - 1)].long()
    s["slots"].copy_(torch.where(live, block * BLOCK + pos % BLOCK, -1))
    s["pos"].copy_(torch.where(live, pos, -1))
    touched = torch.where(n > 0, (total - 1) // BLOCK - length // BLOCK + 1, 0)
    ci = torch.cat([zero, touched.cumsum(0)])
    w = torch.arange(s["items"].shape[0], device=dev)
    r = torch.searchsorted(ci[1:], w, right=True).clamp(max=n.numel() - 1)
    item = torch.stack([r, length[r] // BLOCK + w - ci[r]], 1)
    s["items"].copy_(torch.where((w < ci[-1])[:, None], item, -1))
    s["length_out"].copy_(total)
    s["free_count_out"].copy_(s["free_count"] - cb[-1:])
    s["cu_tokens"].copy_(cu)
    s["cu_blocks"].copy_(cb)
    s["cu_items"].copy_(ci)
    s["status"].copy_(torch.stack([code, cu[-1], ci[-1], cb[-1]]))


def _plain_append(s):
    cu, items = s["cu_tokens"].long(), s["items"].long()
    tokens, kv, d = s["k_new"].shape[0], s["k"].shape[1], s["k"].shape[3]
    r, j = items[:, 0].clamp(min=0), items[:, 1].clamp(min=0)
    total = s["length"].long()[r]
    before = total - (cu[r + 1] - cu[r])
    p = j[:, None] * BLOCK + torch.arange(BLOCK, device=r.device)[None]  # positions of the item's block
    fresh = (p >= before[:, None]) & (p < total[:, None])
    src = (cu[r][:, None] + p - before[:, None]).clamp(0, tokens - 1)
    full = (items[:, 0] >= 0) & (j * BLOCK + BLOCK <= total)
    part = (items[:, 0] >= 0) & ~full
    block = s["table"][r, j.clamp(max=s["table"].shape[1] - 1)].long()
    spare = s["k"].shape[0] - 1  # no request's block: items with nothing to write go there
    block = torch.where(full, block, spare)
    for name, which in (("k", 0), ("v", 1)):
        new = s[name + "_new"].reshape(tokens, kv, d)
        x = torch.where(fresh[:, :, None, None], new[src], s[name + "_tail"][r].transpose(1, 2)).transpose(1, 2)
        codes, scale = _quantise(x.float(), (2, 3), s["code"])
        codes = (codes if which == 0 else _to_v(codes)).view(torch.int8)
        pool = s[name].view(torch.int8)
        keep = full[:, None, None, None]
        pool.index_copy_(0, block, torch.where(keep, codes, pool[spare][None]))
        s["scales"][:, :, which].index_copy_(0, block, torch.where(full[:, None], scale, s["scales"][spare, :, which][None]))
        # a partial block is its request's tail; of a request's items at most one is
        tail = torch.zeros_like(s[name + "_tail"]).index_add_(0, r, torch.where(part[:, None, None, None], x, 0))
        row = torch.zeros((s["length"].numel(), BLOCK), dtype=torch.int32, device=r.device)
        row = row.index_add_(0, r, (fresh & part[:, None]).to(torch.int32)) > 0
        s[name + "_tail"].copy_(torch.where(row[:, None, :, None], tail, s[name + "_tail"]))


def _plain_attend(s):
    cu, length = s["cu_tokens"].long(), s["length"].long()
    tokens, heads, d = s["q"].shape
    reqs, kv, most = length.numel(), s["k"].shape[1], s["most_new"]
    dev = cu.device
    table = s["table"][:, : _blocks(s["most_len"])].long().clamp(min=0)
    j = torch.arange(table.shape[1], device=dev)
    in_tail = (j[None] == (length // BLOCK)[:, None])[:, :, None, None, None]
    scale = s["scales"][table][..., None, None, :]
    k = torch.where(in_tail, s["k_tail"].float()[:, None], _pick(s["k"], table).float() * scale[..., 0])
    v = torch.where(in_tail, s["v_tail"].float()[:, None], _from_v(_pick(s["v"], table)) * scale[..., 1])
    k, v = (x.transpose(1, 2).reshape(reqs, kv, -1, d) for x in (k, v))  # (requests, kv heads, keys, d)
    n = cu[1:] - cu[:-1]
    i = torch.arange(most, device=dev)
    at = (cu[:-1, None] + i[None]).clamp(max=tokens - 1)
    q = s["q"].float()[at].view(reqs, most, kv, heads // kv, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(reqs, kv, -1, d)  # rows: (token, head of the group)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    key = torch.arange(k.shape[2], device=dev)
    seen = key[None, None] <= (length - n)[:, None, None] + i[None, :, None]  # (requests, new tokens, keys)
    seen &= (i[None] < n[:, None])[..., None]
    x = x.view(reqs, kv, most, heads // kv, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    x = (x - top).exp_()
    total = x.sum(-1, keepdim=True)
    # a key that no token of the request sees has weight 0; what lies there need not be finite
    v = torch.where((key[None] < length[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(x.view(reqs, kv, -1, k.shape[2]), v).view(reqs, kv, most, -1, d)
    o = (o / total.clamp_min(torch.finfo(torch.float32).tiny)).permute(0, 2, 1, 3, 4).reshape(reqs, most, heads, d)
    t = torch.arange(tokens, device=dev)
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=reqs - 1)
    s["o"].copy_(o[r, t - cu[r]])


def _plain_linear(s):
    m, k = s["x"].shape
    n, kb = s["b"].shape[0], s["a_scales"].shape[1]
    x = torch.zeros((m, kb * GROUP), device=s["x"].device)
    x[:, :k] = s["x"]
    codes, scale = _quantise(x.view(m, kb, GROUP), (2,), "e4m3")
    a = (codes.float() * scale[..., None]).view(m, -1)[:, :k]
    rows = torch.arange(n, device=x.device) // GROUP
    b = s["b"].float() * s["b_scales"][rows].repeat_interleave(GROUP, dim=1)[:, :k]
    s["y"].copy_(torch.matmul(a, b.t().contiguous()))
    s["a"].copy_(codes.view(m, -1)[:, :k])
    s["a_scales"].copy_(scale)


# ---- the framework's calls --------------------------------------------------------------------------


def _own_call(s):
    import tsfm_attn as ta

    kind = s["kind"]
    if kind == "plan":
        rc = ta.kv8_plan(s["n_new"], s["length"], s["length_out"], s["free_list"], s["free_count"], s["free_count_out"],
                         s["table"], s["cu_tokens"], s["cu_blocks"], s["cu_items"], s["slots"], s["pos"], s["items"], s["status"])
    elif kind == "append":
        rc = ta.kv8_append(s["cache"], s["k_new"], s["v_new"], s["cu_tokens"], s["items"])
    elif kind == "attend":
        rc = ta.kv8_attend(s["cache"], s["q"], s["o"], s["cu_tokens"], scale=s["scale"], max_new=s["most_new"],
                           max_len=s["most_len"], workspace=s["workspace"])
    else:
        rc = ta.f8_quantize(s["x"], s["a"], s["a_scales"])
        rc = rc or ta.f8_gemm_nt(s["a"], s["a_scales"], s["b"], s["b_scales"], s["y"])
    if rc != ta.OK:
        raise ta.TsfmError(rc, ta.last_error())


def run(state):
    kind = state["kind"]
    if own:
        _own_call(state)
    else:
        {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "linear": _plain_linear}[kind](state)
    names = {"plan": ("table", "length_out", "free_count_out", "cu_tokens", "cu_blocks", "cu_items", "slots", "pos",
                      "items", "status"),
             "append": ("k", "v", "scales", "k_tail", "v_tail"), "attend": ("o",), "linear": ("a", "a_scales", "y")}[kind]
    return {n: state[n] for n in names}


# ---- the definitions in float64 ---------------------------------------------------------------------


def _e4m3_values():
    """The non-negative e4m3 values, by code: 3 bits of mantissa, 4 of exponent with bias 7, subnormals."""
    v = [(c & 7) * 2.0 ** -9 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)]
    return torch.tensor(v, dtype=torch.float64, device="cuda")


def _nearest_e4m3(x):
    """x (float64, |x| <= 448) to the nearest e4m3 value, the even code where two are as near."""
    grid = _e4m3_values()
    mid = (grid[1:] + grid[:-1]) / 2
    low = torch.searchsorted(mid, x.abs().contiguous())  # values up to and at a midpoint go to the code below it
    tie = (low < 126) & (x.abs() == mid[low.clamp(max=125)]) & (low % 2 == 1)
    return torch.sign(x) * grid[(low + tie).clamp(max=126)]


def _exact_scale(amax):
    e = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -140) / E4M3_MAX)).long()
    s = ((e + 1023) << 52).view(torch.float64)  # its bits: a power function need not be exact
    s = torch.where(amax > E4M3_MAX * s, 2 * s, torch.where(amax <= E4M3_MAX * s / 2, s / 2, s))
    return torch.where(amax > 0, s.clamp_min(2.0 ** -126), torch.ones_like(s))


def _exact_append(s):
    cu, total, items = s["cu_tokens"].tolist(), s["length"].tolist(), s["items"].tolist()
    table, tails = s["table"].tolist(), {n: s[n + "_tail"].double() for n in ("k", "v")}
    out = {"k": s["k"].double(), "v": s["v"].double(), "scales": s["scales"].double()}
    kv, d = s["k"].shape[1], s["k"].shape[3]
    order = torch.tensor([32 * (b // 8 % 2) + 16 * (b // 4 % 2) + 4 * (b // 16) + b % 4 for b in range(BLOCK)], device="cuda")
    old = {n: t.clone() for n, t in tails.items()}
    for r, j in items:
        if r < 0:
            continue
        before = total[r] - (cu[r + 1] - cu[r])
        lo, hi = max(before, j * BLOCK), min(total[r], j * BLOCK + BLOCK)
        a = cu[r] + lo - before
        for which, n in enumerate(("k", "v")):
            x = s[n + "_new"][a:a + hi - lo].double().reshape(hi - lo, kv, d).transpose(0, 1)
            if hi < j * BLOCK + BLOCK:
                tails[n][r, :, lo % BLOCK:lo % BLOCK + hi - lo] = x
                continue
            x = torch.cat([old[n][r, :, : lo - j * BLOCK], x], dim=1)
            amax = x.abs().amax(dim=(1, 2))
            if s["code"] == "e4m3":
                scale = _exact_scale(amax)
                codes = _nearest_e4m3(x / scale[:, None, None])
                out[n][table[r][j]] = codes if n == "k" else codes.transpose(1, 2)[:, :, order]
            else:
                scale = torch.where(amax > 0, amax.clamp_min(2.0 ** -100) / 127, 1.0)
            out["scales"][table[r][j], :, which] = scale
    if s["code"] != "e4m3":  # a whole number has no value in 64 bits: where it rounds from is 32-bit arithmetic
        out["k"] = out["v"] = None
    return {**out, "k_tail": tails["k"], "v_tail": tails["v"]}


def _exact_attend(s):
    cu, total = s["cu_tokens"].tolist(), s["length"].tolist()
    tokens, heads, d = s["q"].shape
    kv = s["k"].shape[1]
    byte = torch.tensor([16 * (t // 4 % 4) + 8 * (t // 32) + 4 * (t // 16 % 2) + t % 4 for t in range(BLOCK)], device="cuda")
    out = torch.empty((tokens, heads, d), dtype=torch.float64, device="cuda")
    for r, length in enumerate(total):
        n = cu[r + 1] - cu[r]
        if n == 0:
            continue
        ids = s["table"][r, : length // BLOCK].long()
        for h in range(kv):
            sc = s["scales"][ids, h].double()
            k = (_pick(s["k"], ids, h).double() * sc[:, 0, None, None]).reshape(-1, d)
            v = (_pick(s["v"], ids, h).double()[:, :, byte] * sc[:, 1, None, None]).transpose(1, 2).reshape(-1, d)
            rest = length % BLOCK
            k = torch.cat([k, s["k_tail"][r, h, :rest].double()])
            v = torch.cat([v, s["v_tail"][r, h, :rest].double()])
            for at in range(0, n, 512):
                m = min(512, n - at)
                g = heads // kv
                q = s["q"][cu[r] + at:cu[r] + at + m, h * g:(h + 1) * g].double().reshape(m * g, d)
                x = q @ k.t() * s["scale"]
                last = length - n + at + torch.arange(m, device="cuda").repeat_interleave(g)
                x = x.masked_fill(torch.arange(length, device="cuda")[None] > last[:, None], -math.inf)
                out[cu[r] + at:cu[r] + at + m, h * g:(h + 1) * g] = (torch.softmax(x, -1) @ v).view(m, g, d)
    return {"o": out}


def _exact_linear(s):
    m, k = s["x"].shape
    n, kb = s["b"].shape[0], s["a_scales"].shape[1]
    codes = torch.empty((m, k), dtype=torch.float64, device="cuda")
    scales = torch.empty((m, kb), dtype=torch.float64, device="cuda")
    y = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    for g in range(kb):
        part = slice(g * GROUP, min(k, g * GROUP + GROUP))
        x = s["x"][:, part].double()
        scales[:, g] = _exact_scale(x.abs().amax(dim=1))
        codes[:, part] = _nearest_e4m3(x / scales[:, g, None])
        b = s["b"][:, part].double() * s["b_scales"][:, g].double().repeat_interleave(GROUP)[:n, None]
        y += (codes[:, part] * scales[:, g, None]) @ b.t()
    return {"a": codes, "a_scales": scales, "y": y}


def exact(case, seed):
    if case["kind"] == "plan":  # whole numbers only
        return None
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "linear": _exact_linear}[case["kind"]](s)
