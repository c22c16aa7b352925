"""The paged 8-bit K/V cache and its attention (tsfm_kv8_*) against plain models: block tables and slot maps, the
cache's bytes, attention against float64 with bounds from the roundings that are made, and what lies at the edges:
requests without tokens, lengths around a block, values that are no numbers, tables that name no block, captured
steps, streams, pools past 4 GiB."""
import numpy as np
import pytest

import _kv8_ref as ref

pytestmark = pytest.mark.gpu

HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative: torch.finfo(t).eps / 2


def _t():
    import torch

    return torch


def _dtype(name):
    return _t().bfloat16 if name == "bf16" else _t().float16


def _round(x, name):
    """f32 numpy values as the 16-bit type holds them."""
    return _t().from_numpy(np.ascontiguousarray(x, np.float32)).to(_dtype(name)).float().numpy()


def _dev(x, name):
    return _t().from_numpy(np.ascontiguousarray(x, np.float32)).to(_dtype(name)).cuda()


def _pool(ta, requests, blocks, kv, d, code, dtype, max_len, max_tokens):
    torch = _t()
    p = ta.Kv8Pool(requests, blocks, kv, d, max_len=max_len, max_tokens=max_tokens, dtype=_dtype(dtype),
                   code=ta.CODE_E4M3 if code == "e4m3" else ta.CODE_I8)
    # What nothing wrote must not matter: NaN codes (or the largest), NaN scales, NaN tails.
    p.cache.k.view(torch.uint8).fill_(0x7f)
    p.cache.v.view(torch.uint8).fill_(0x7f)
    p.cache.scales.fill_(float("nan"))
    p.cache.k_tail.fill_(float("nan"))
    p.cache.v_tail.fill_(float("nan"))
    return p


def _tokens(rng, n, kv, d, dtype, loud=4.0):
    x = rng.standard_normal((n, kv, d)).astype(np.float32)
    x[:, :, ::17] *= loud
    return _round(x, dtype)


def _step(torch, pool, model, n_new, k, v, dtype):
    """Plans and appends the packed tokens, on the GPU and in the model; checks the plan."""
    total, room = sum(max(0, n) for n in n_new), pool.slots.numel()
    want = model.plan(n_new)
    pool.step(torch.tensor(n_new, dtype=torch.int32, device="cuda"))
    row = k.shape[1] * k.shape[2]
    kd, vd = _dev(k.reshape(total, row), dtype), _dev(v.reshape(total, row), dtype)
    if total:
        pool.append(kd, vd)
    model.append(n_new, k, v)
    cu, cb, ci, slots, pos, items = want
    assert pool.status.tolist() == [0, total, len(items), cb[-1]]
    assert pool.cu_tokens.tolist() == cu and pool.cu_blocks.tolist() == cb and pool.cu_items.tolist() == ci
    assert pool.slots.tolist() == slots + [-1] * (room - total)
    assert pool.pos.tolist() == pos + [-1] * (room - total)
    assert [tuple(i) for i in pool.items.tolist()] == items + [(-1, -1)] * (pool.items.shape[0] - len(items))
    assert pool.length.tolist() == model.lengths()
    assert pool.free_count.item() == len(model.free) and pool.free_list[:len(model.free)].tolist() == model.free
    for r, row in enumerate(pool.table.tolist()):
        assert row == model.table[r] + [-1] * (len(row) - len(model.table[r]))


def _check_bytes(torch, pool, model, kv):
    """Every whole block's codes and scales, and every tail, hold exactly what the model says."""
    k = pool.cache.k.view(torch.uint8).cpu().numpy()
    v = pool.cache.v.view(torch.uint8).cpu().numpy()
    s = pool.cache.scales.cpu().numpy()
    kt, vt = pool.cache.k_tail.float().cpu().numpy(), pool.cache.v_tail.float().cpu().numpy()
    for r, n in enumerate(model.lengths()):
        for j in range(n // 64):
            b = model.table[r][j]
            for h in range(kv):
                for which, got in ((0, k[b, h]), (1, v[b, h].T[ref.V_BYTE])):
                    codes, scale = model.block(r, j, h, which)
                    assert np.array_equal(s[b, h, which], scale, equal_nan=True), (r, j, h, which)
                    assert np.array_equal(got, codes), (r, j, h, which)
        rest = n % 64
        for got, x in ((kt, model.k[r]), (vt, model.v[r])):
            assert np.array_equal(got[r, :, :rest], x[n - rest:].transpose(1, 0, 2), equal_nan=True), r


def _check_attend(torch, pool, model, n_new, q, o, scale, dtype, kv, skip=()):
    """o's rows against float64, request by request; bounds as attend_bound derives them."""
    heads = q.shape[1]
    at = 0
    got = o.float().cpu().numpy().astype(np.float64)
    for r, n in enumerate(n_new):
        n = max(0, n)
        if n and r not in skip:
            length = len(model.k[r])
            last = length - n + np.arange(n)
            for h in range(kv):
                k, v = model.values(r, h)
                for hq in range(h * heads // kv, (h + 1) * heads // kv):
                    want, a, s = ref.attend(q[at:at + n, hq], k, v, last, scale)
                    bound = ref.attend_bound(want, a, s, np.abs(v).max(), length, HALF[dtype], dtype == "f16")
                    err = np.abs(got[at:at + n, hq] - want)
                    assert (err <= bound).all(), (r, hq, float((err / bound).max()))
        at += n


CACHES = [("e4m3", "bf16", 64, 4, 4), ("e4m3", "f16", 128, 6, 2), ("i8", "bf16", 128, 8, 1), ("i8", "f16", 64, 6, 2),
          ("e4m3", "bf16", 128, 3, 3), ("i8", "f16", 128, 64, 1)]


@pytest.mark.parametrize("code,dtype,d,heads,kv", CACHES)
def test_steps_match_the_model(ta, gpu_ready, code, dtype, d, heads, kv):
    """Prompts, single tokens and blocks of 32 in turn, lengths on both sides of every block edge, requests that get
    nothing: plan, bytes of the cache and attention after every step."""
    torch = _t()
    rng = np.random.default_rng(7)
    R, room = 6, 700
    pool = _pool(ta, R, 40, kv, d, code, dtype, 1024, room)
    model = ref.Model(R, kv, d, code, 40, 16)
    steps = [[63, 64, 65, 0, 1, 200], [1, 1, 1, 0, 1, 1], [1, 0, 1, -3, 62, 1], [70, 32, 32, 32, 1, 130],
             [1, 1, 1, 1, 1, 1], [0, 0, 0, 0, 0, 0], [129, 63, 0, 300, 2, 1]]
    for n_new in steps:
        total = sum(max(0, n) for n in n_new)
        k, v = _tokens(rng, total, kv, d, dtype), _tokens(rng, total, kv, d, dtype, 1.0)
        q = _round(rng.standard_normal((total, heads, d)), dtype)
        _step(torch, pool, model, n_new, k, v, dtype)
        _check_bytes(torch, pool, model, kv)
        qd = _dev(np.concatenate([q, np.zeros((5, heads, d), np.float32)]), dtype)
        o = torch.full((total + 5, heads, d), -7.0, dtype=_dtype(dtype), device="cuda")
        pool.attend(qd, o, d ** -0.5, max_new=max(n_new), max_len=max(model.lengths()))
        assert (o[total:] == -7).all()  # rows behind the last token
        _check_attend(torch, pool, model, n_new, q, o, d ** -0.5, dtype, kv)


@pytest.mark.parametrize("code,dtype", [("e4m3", "bf16"), ("i8", "f16")])
def test_cache_does_not_depend_on_the_calls(ta, gpu_ready, code, dtype):
    """200 tokens in one call, one by one, and in unequal pieces (some complete an old block and leave a new tail in
    one call): the same bytes."""
    torch = _t()
    rng = np.random.default_rng(3)
    kv, d, n = 2, 64, 200
    k, v = _tokens(rng, n, kv, d, dtype), _tokens(rng, n, kv, d, dtype)
    seen = []
    for pieces in ([200], [1] * 200, [70, 60, 69, 1], [3, 130, 60, 7], [64, 64, 64, 8]):
        pool = _pool(ta, 1, 4, kv, d, code, dtype, 256, 256)
        model = ref.Model(1, kv, d, code, 4, 4)
        at = 0
        for p in pieces:
            _step(torch, pool, model, [p], k[at:at + p], v[at:at + p], dtype)
            at += p
        _check_bytes(torch, pool, model, kv)
        t = pool.table[0, :3].long()
        seen.append([pool.cache.k.view(torch.uint8)[t], pool.cache.v.view(torch.uint8)[t], pool.cache.scales[t],
                     pool.cache.k_tail[:, :, :8], pool.cache.v_tail[:, :, :8]])
    for other in seen[1:]:
        for a, b in zip(seen[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("code,dtype", [("e4m3", "bf16"), ("e4m3", "f16"), ("i8", "bf16"), ("i8", "f16")])
def test_blocks_of_any_size_of_value(ta, gpu_ready, code, dtype):
    """Blocks of zeros, of the type's smallest and largest values, of one large value among small ones, of both zeros
    and midpoints between codes."""
    torch = _t()
    kv, d = 1, 64
    rng = np.random.default_rng(5)
    fin = torch.finfo(_dtype(dtype))
    x = np.zeros((8 * 64, kv, d), np.float32)
    x[64:128] = fin.tiny * rng.choice([-1, 1], (64, kv, d))
    x[128:192] = fin.max * rng.choice([-1, 1], (64, kv, d))
    x[192:256] = rng.standard_normal((64, kv, d)) * 1e-3
    x[200, 0, 3] = 900.0
    x[256:320] = rng.choice([-0.0, 0.0, 17.0, 19.0, 21.0, 0.00146484375, 448.0], (64, kv, d))
    x[320:384] = rng.standard_normal((64, kv, d)) * fin.tiny * 4
    x[384:448] = rng.integers(-127, 128, (64, kv, d)) + 0.5
    x[448:] = rng.standard_normal((64, kv, d))
    x = _round(x, dtype)
    pool = _pool(ta, 1, 8, kv, d, code, dtype, 512, 512)
    model = ref.Model(1, kv, d, code, 8, 8)
    _step(torch, pool, model, [512], x, x[::-1].copy(), dtype)
    _check_bytes(torch, pool, model, kv)


@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2), (3, 1)])
@pytest.mark.parametrize("lens,news", [
    ([1], [1]), ([64], [1]), ([65], [1]), ([700, 1, 130], [1, 1, 1]), ([300, 64], [32, 32]), ([257, 90, 640], [17, 90, 200]),
    ([2000, 33], [1, 33])])
@pytest.mark.parametrize("code,dtype,d", [("e4m3", "bf16", 64), ("i8", "f16", 128)])
def test_attend_shapes(ta, gpu_ready, code, dtype, d, heads, kv, lens, news):
    """Lengths, new tokens and head groups of every kernel and split; the hints absent, right and wrong."""
    torch = _t()
    rng = np.random.default_rng(sum(lens) + heads)
    R, total = len(lens), sum(news)
    pool = _pool(ta, R, sum(-(-n // 64) for n in lens), kv, d, code, dtype, 4096, sum(lens) + 1)
    model = ref.Model(R, kv, d, code, pool.cache.blocks, 64)
    for n_new in ([n - m for n, m in zip(lens, news)], news):
        t = sum(n_new)
        _step(torch, pool, model, n_new, _tokens(rng, t, kv, d, dtype), _tokens(rng, t, kv, d, dtype, 1.0), dtype)
    q = _round(rng.standard_normal((total, heads, d)) * 2, dtype)
    qd = _dev(q, dtype)
    for new, length in ((max(news), max(lens)), (0, 0), (1, 1), (max(news), 100), (4096, 1 << 20)):
        o = torch.empty_like(qd)
        pool.attend(qd, o, d ** -0.5, max_new=new, max_len=length)
        _check_attend(torch, pool, model, news, q, o, d ** -0.5, dtype, kv)


@pytest.mark.parametrize("code,dtype", [("e4m3", "f16"), ("i8", "bf16")])
@pytest.mark.parametrize("news", [[1, 1], [40, 64]])
def test_attend_scales_and_scores(ta, gpu_ready, code, dtype, news):
    """Blocks whose values differ by 10^6 between them (K and V), scores that keep rising along the keys, scale 1 and
    0: the weights carry the V scale, and lose nothing by it."""
    torch = _t()
    rng = np.random.default_rng(11)
    kv, heads, d, n = 2, 4, 64, 640
    pool = _pool(ta, 2, 24, kv, d, code, dtype, 1024, 2 * n + 1)
    model = ref.Model(2, kv, d, code, 24, 16)
    total = 2 * n
    k, v = _tokens(rng, total, kv, d, dtype), _tokens(rng, total, kv, d, dtype, 1.0)
    k *= np.tile(np.linspace(0.1, 3.0, n), 2)[:, None, None].astype(np.float32)
    v *= np.repeat(10.0 ** rng.integers(-3, 4, 2 * n // 64), 64)[:, None, None].astype(np.float32)
    v[n:] = v[n:][::-1]
    k, v = _round(k, dtype), _round(v, dtype)
    first = [n - m for m in news]
    keep = np.concatenate([np.arange(first[0]), n + np.arange(first[1])])
    rest = np.concatenate([np.arange(first[0], n), n + np.arange(first[1], n)])
    _step(torch, pool, model, first, k[keep], v[keep], dtype)
    _step(torch, pool, model, news, k[rest], v[rest], dtype)
    q = _round(rng.standard_normal((sum(news), heads, d)), dtype)
    qd = _dev(q, dtype)
    for scale in (0.125, 1.0, 0.0):
        o = torch.empty_like(qd)
        pool.attend(qd, o, scale, max_new=max(news), max_len=n)
        _check_attend(torch, pool, model, news, q, o, scale, dtype, kv)


@pytest.mark.parametrize("news", [1, 20, 100])
@pytest.mark.parametrize("code,dtype,d", [("e4m3", "bf16", 64), ("i8", "f16", 128)])
def test_values_that_are_no_numbers(ta, gpu_ready, code, dtype, d, news):
    """A NaN or infinity in a tail's V reaches the rows that read its token and no other; in a whole block, K's or V's,
    the rows that read the block; another request never."""
    torch = _t()
    rng = np.random.default_rng(13)
    kv = heads = 2
    held = 128 - news % 64 + 40  # the last tokens lie in the tail
    n = held + news
    for bad in (float("nan"), float("inf"), -float("inf")):
        for where in ("v_tail", "k_block", "v_block"):
            pool = _pool(ta, 2, 12, kv, d, code, dtype, 512, 2 * n + 1)
            model = ref.Model(2, kv, d, code, 12, 8)
            k, v = _tokens(rng, 2 * n, kv, d, dtype), _tokens(rng, 2 * n, kv, d, dtype)
            q = _round(rng.standard_normal((2 * news, heads, d)), dtype)
            tok = n - 1 if where == "v_tail" else 5
            (k if where == "k_block" else v)[tok, 1, 3] = bad  # of request 0, head 1
            assert where != "v_tail" or tok >= n // 64 * 64
            keep = np.concatenate([np.arange(held), n + np.arange(held)])
            rest = np.concatenate([np.arange(held, n), n + np.arange(held, n)])
            _step(torch, pool, model, [held, held], k[keep], v[keep], dtype)
            _step(torch, pool, model, [news, news], k[rest], v[rest], dtype)
            o = torch.empty((2 * news, heads, d), dtype=_dtype(dtype), device="cuda")
            pool.attend(_dev(q, dtype), o, d ** -0.5, max_new=news, max_len=n)
            isnan = torch.isnan(o).all(-1).cpu().numpy()
            want = np.zeros((2 * news, heads), bool)
            want[:news, 1] = where != "v_tail"
            want[news - 1, 1] = True
            assert np.array_equal(isnan, want), (bad, where)
            assert torch.isfinite(o[torch.from_numpy(~want).cuda()]).all()
            # the rows without it are what they are without it
            clean_k, clean_v = k.copy(), v.copy()
            (clean_k if where == "k_block" else clean_v)[tok, 1, 3] = 0
            if where == "v_tail" and news > 1:
                model.v[0][tok, 1, 3] = 0
                got = o.clone()
                got[news - 1, 1] = 0
                kk, vv = model.values(0, 1)
                w, a, s = ref.attend(q[:news - 1, 1], kk, vv, held + np.arange(news - 1), d ** -0.5)
                b = ref.attend_bound(w, a, s, np.abs(vv).max(), n, HALF[dtype], dtype == "f16")
                assert (np.abs(got[:news - 1, 1].float().cpu().numpy() - w) <= b).all()


def test_tail_k_that_is_masked(ta, gpu_ready):
    """An infinite K of a later token of the same step: the earlier rows do not see it."""
    torch = _t()
    rng = np.random.default_rng(17)
    for code, dtype, news in (("e4m3", "bf16", 7), ("i8", "f16", 40)):
        pool = _pool(ta, 1, 4, 1, 64, code, dtype, 256, 256)
        model = ref.Model(1, 1, 64, code, 4, 4)
        k, v = _tokens(rng, news, 1, 64, dtype), _tokens(rng, news, 1, 64, dtype)
        k[-1, 0, 0] = float("inf")
        _step(torch, pool, model, [news], k, v, dtype)
        q = _round(rng.standard_normal((news, 1, 64)), dtype)
        o = torch.empty((news, 1, 64), dtype=_dtype(dtype), device="cuda")
        pool.attend(_dev(q, dtype), o, 0.125, max_new=news, max_len=news)
        want, a, s = ref.attend(q[:-1, 0], k[:-1, 0], v[:-1, 0], np.arange(news - 1), 0.125)
        b = ref.attend_bound(want, a, s, np.abs(v).max(), news, HALF[dtype], dtype == "f16")
        assert (np.abs(o[:-1, 0].float().cpu().numpy() - want) <= b).all()


@pytest.mark.parametrize("why,n_new", [(1, [40, 30, 0]), (2, [0, 0, 65]), (3, [64, 0, 3])])
def test_step_that_cannot_be_served(ta, gpu_ready, why, n_new):
    """Too many tokens, a request past its table row, too few blocks: the reason in status, nothing moves, and the
    step's other calls do nothing."""
    torch = _t()
    rng = np.random.default_rng(19)
    pool = _pool(ta, 3, 2, 1, 64, "e4m3", "bf16", 64, 69)
    model = ref.Model(3, 1, 64, "e4m3", 2, 1)
    k = _tokens(rng, 70, 1, 64, "bf16")
    _step(torch, pool, model, [0, 1, 0], k[:1], k[:1], "bf16")
    before = {n: getattr(pool, n).clone() for n in ("length", "table", "free_list", "free_count")}
    cache = [t.clone() for t in (pool.cache.k.view(torch.uint8), pool.cache.v.view(torch.uint8), pool.cache.k_tail)]
    pool.step(torch.tensor(n_new, dtype=torch.int32, device="cuda"))
    assert pool.status.tolist() == [why, 0, 0, 0]
    for n, t in before.items():
        assert torch.equal(getattr(pool, n), t), n
    assert pool.cu_tokens.tolist() == [0] * 4 and (pool.slots == -1).all() and (pool.items == -1).all()
    x = _dev(k.reshape(70, 64), "bf16")
    pool.append(x, x)
    o = torch.full((70, 1, 64), -7.0, dtype=torch.bfloat16, device="cuda")
    pool.attend(x.view(70, 1, 64), o, 0.125)
    assert (o == -7).all()
    for a, b in zip(cache, (pool.cache.k.view(torch.uint8), pool.cache.v.view(torch.uint8), pool.cache.k_tail)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_negative_lengths_and_counts(ta, gpu_ready):
    """A negative length cannot be served; a free count past the pool is taken as the pool."""
    torch = _t()
    pool = _pool(ta, 2, 4, 1, 64, "i8", "f16", 128, 8)
    pool.length[1] = -5
    pool.step(torch.tensor([1, 1], dtype=torch.int32, device="cuda"))
    assert pool.status.tolist() == [2, 0, 0, 0] and pool.length.tolist() == [0, -5]
    pool.length[1] = 0
    pool.free_count.fill_(1000)
    pool.step(torch.tensor([1, 1], dtype=torch.int32, device="cuda"))
    assert pool.status.tolist() == [0, 2, 2, 2] and pool.free_count.item() == 2


@pytest.mark.parametrize("R,most", [(1, 3000), (700, 3), (1024, 40), (1025, 2), (5000, 1), (3, 20000)])
def test_plan_of_many(ta, gpu_ready, R, most):
    """More requests than a round of the scan takes, more tokens than a workgroup maps, long requests, most of them
    without tokens: against the model."""
    torch = _t()
    rng = np.random.default_rng(R)
    n1, n2 = ([int(n) for n in rng.integers(0, most + 1, R) * (rng.random(R) < 0.6)] for _ in range(2))
    room = max(sum(n1), sum(n2)) + 77
    width = -(-2 * most // 64) + 1
    blocks = sum(-(-(a + b) // 64) for a, b in zip(n1, n2)) + 3
    pool = _pool(ta, R, blocks, 1, 64, "e4m3", "bf16", width * 64, room)
    model = ref.Model(R, 1, 64, "e4m3", blocks, width)
    for n_new in (n1, n2):
        z = np.zeros((sum(n_new), 1, 64), np.float32)
        _step(torch, pool, model, n_new, z, z, "bf16")


def test_plan_out_of_place(ta, gpu_ready):
    """len_out and free_count_out apart from their inputs: the inputs stay, and the plan can be made again."""
    torch = _t()

    def ints(*v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    length, free_count, free_list = ints(10, 64, 0), ints(5), ints(0, 1, 2, 3, 4, -9)
    table = torch.full((3, 3), -1, dtype=torch.int32, device="cuda")
    table[0, 0], table[1, 0] = 9, 8  # (a pool of 6 blocks: ids are not checked here)
    for _ in range(2):
        out = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (3, 1, 4, 4, 4)]
        slots, pos = torch.empty(9, dtype=torch.int64, device="cuda"), torch.empty(9, dtype=torch.int32, device="cuda")
        items, status = torch.empty((9, 2), dtype=torch.int32, device="cuda"), ints(9, 9, 9, 9)
        assert ta.kv8_plan(ints(2, 3, 1), length, out[0], free_list, free_count, out[1], table, *out[2:], slots, pos,
                           items, status) == ta.OK
        assert length.tolist() == [10, 64, 0] and free_count.item() == 5
        assert out[0].tolist() == [12, 67, 1] and out[1].item() == 3
        assert table.tolist() == [[9, -1, -1], [8, 4, -1], [3, -1, -1]]
        assert slots.tolist() == [9 * 64 + 10, 9 * 64 + 11, 256, 257, 258, 192, -1, -1, -1]
        assert pos.tolist() == [10, 11, 64, 65, 66, 0, -1, -1, -1]


def test_release_and_reuse(ta, gpu_ready):
    """Ended requests' blocks serve the next ones; a list that would pass the pool is refused."""
    torch = _t()
    rng = np.random.default_rng(23)
    R, kv, d = 1500, 1, 64
    pool = _pool(ta, R, 1600, kv, d, "i8", "bf16", 512, 4000)
    model = ref.Model(R, kv, d, "i8", 1600, 8)
    for _ in range(4):
        n_new = [int(n) for n in rng.integers(0, 200, R) * (rng.random(R) < 0.02)]
        t = sum(n_new)
        _step(torch, pool, model, n_new, _tokens(rng, t, kv, d, "bf16"), _tokens(rng, t, kv, d, "bf16"), "bf16")
        drop = (rng.random(R) < 0.4).astype(np.uint8)
        freed = sum(len(model.table[r]) for r in range(R) if drop[r])
        pool.release(torch.from_numpy(drop).cuda())
        model.release(drop)
        assert pool.status[:2].tolist() == [0, freed]
        assert pool.free_count.item() == len(model.free)
        assert pool.free_list[:len(model.free)].tolist() == model.free
        assert pool.length.tolist() == model.lengths()
        assert [[i for i in row if i >= 0] for row in pool.table.tolist()] == model.table
        _check_bytes(torch, pool, model, kv)
    drop = torch.ones(R, dtype=torch.uint8, device="cuda")
    n = [5] + [0] * (R - 1)
    _step(torch, pool, model, n, _tokens(rng, 5, kv, d, "bf16"), _tokens(rng, 5, kv, d, "bf16"), "bf16")
    pool.free_count.fill_(1600)
    before = [pool.length.clone(), pool.table.clone(), pool.free_list.clone()]
    pool.release(drop)
    assert pool.status[:2].tolist() == [1, 0] and pool.free_count.item() == 1600
    for a, b in zip(before, (pool.length, pool.table, pool.free_list)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("entry", [-1, 12, 1 << 30, -(1 << 31)])
def test_table_entries_that_are_no_block(ta, gpu_ready, entry):
    """A table that names no block: the rows that read there become NaN, others are right, and nothing is written."""
    torch = _t()
    rng = np.random.default_rng(29)
    kv, d, dtype = 2, 64, "bf16"
    for news in ([1, 1], [33, 60]):
        pool = _pool(ta, 2, 12, kv, d, "e4m3", dtype, 512, 400)
        model = ref.Model(2, kv, d, "e4m3", 12, 8)
        first = [150, 130]
        t = sum(first)
        _step(torch, pool, model, first, _tokens(rng, t, kv, d, dtype), _tokens(rng, t, kv, d, dtype), dtype)
        t = sum(news)
        _step(torch, pool, model, news, _tokens(rng, t, kv, d, dtype), _tokens(rng, t, kv, d, dtype), dtype)
        pool.table[0, 1] = entry
        q = _round(rng.standard_normal((t, kv, d)), dtype)
        o = torch.empty((t, kv, d), dtype=torch.bfloat16, device="cuda")
        pool.attend(_dev(q, dtype), o, 0.125, max_new=max(news), max_len=256)
        assert torch.isnan(o[:news[0]]).all()
        _check_attend(torch, pool, model, news, q, o, 0.125, dtype, kv, skip=(0,))
        # the block that a step completes there is not written
        before = [x.clone() for x in (pool.cache.k.view(torch.uint8), pool.cache.v.view(torch.uint8), pool.cache.scales)]
        more = 192 - int(pool.length[0]) % 192
        pool.step(torch.tensor([more, 0], dtype=torch.int32, device="cuda"))
        pool.table[0, 2] = entry
        x = _dev(rng.standard_normal((more, kv * d)), dtype)
        pool.append(x, x)
        full = int(pool.length[0]) // 64
        keep = [b for b in range(12) if b not in pool.table[0, 3:full].tolist()]
        for a, b in zip(before, (pool.cache.k.view(torch.uint8), pool.cache.v.view(torch.uint8), pool.cache.scales)):
            assert torch.equal(a[keep].view(torch.uint8), b[keep].view(torch.uint8))


def test_counts_that_do_not_fit(ta, gpu_ready):
    """Prefix sums past the packed rows, decreasing ones, lengths past the table or below the new tokens, items of no
    request: every access stays in the arrays, rows without keys are 0 (the counts are clamped)."""
    torch = _t()
    rng = np.random.default_rng(31)
    kv, d, dtype, T = 2, 64, "bf16", 80
    pool = _pool(ta, 3, 12, kv, d, "i8", dtype, 256, 80)
    model = ref.Model(3, kv, d, "i8", 12, 4)
    k = _tokens(rng, T, kv, d, dtype)
    _step(torch, pool, model, [40, 30, 10], k, k, dtype)
    q, o = _dev(rng.standard_normal((T, kv, d)), dtype), torch.full((T, kv, d), -7.0, dtype=torch.bfloat16, device="cuda")
    big = (1 << 31) - 1
    for cu, length in (([0, 1000, 2000, big], [40, 30, 10]), ([-5, 90, 20, 10], [40, 30, 10]),
                       ([0, 40, 70, 80], [big, 30, 10]), ([0, 40, 70, 80], [-3, 30, 10])):
        pool.cu_tokens.copy_(torch.tensor(cu, dtype=torch.int32))
        pool.length.copy_(torch.tensor(length, dtype=torch.int32))
        pool.items[:4] = torch.tensor([[5, 0], [-1, 3], [0, 77], [big, big]], dtype=torch.int32)
        x = _dev(k.reshape(T, -1), dtype)
        pool.append(x, x)
        for new in (1, 80):
            pool.attend(q, o, 0.125, max_new=new)
    # a request shorter than its new tokens: the rows before its start read nothing
    pool.cu_tokens.copy_(torch.tensor([0, 40, 70, 80], dtype=torch.int32))
    pool.length.copy_(torch.tensor([25, 30, 10], dtype=torch.int32))
    for new in (1, 80):
        o.fill_(-7)
        pool.attend(q, o, 0.125, max_new=new)
        assert (o[:15] == 0).all() and (o[15:40] != 0).any()


def test_views_and_strides(ta, gpu_ready):
    """k, v and q as parts of one fused projection, o as part of a wider row: the neighbours stay."""
    torch = _t()
    rng = np.random.default_rng(37)
    kv, heads, d, dtype, n = 2, 4, 128, "f16", 90
    pool = _pool(ta, 1, 4, kv, d, "e4m3", dtype, 256, n)
    model = ref.Model(1, kv, d, "e4m3", 4, 4)
    qkv = _round(rng.standard_normal((n, (heads + 2 * kv) * d)), dtype)
    dev = _dev(qkv, dtype)
    q, k, v = dev[:, :heads * d], dev[:, heads * d:(heads + kv) * d], dev[:, (heads + kv) * d:]
    model.plan([n])
    pool.step(torch.tensor([n], dtype=torch.int32, device="cuda"))
    pool.append(k, v)
    model.append([n], qkv[:, heads * d:(heads + kv) * d].reshape(n, kv, d), qkv[:, (heads + kv) * d:].reshape(n, kv, d))
    _check_bytes(torch, pool, model, kv)
    wide = torch.full((n, heads * d + 24), -7.0, dtype=torch.float16, device="cuda")
    pool.attend(q, wide[:, 8:8 + heads * d], d ** -0.5)
    assert (wide[:, :8] == -7).all() and (wide[:, 8 + heads * d:] == -7).all()
    o = wide[:, 8:8 + heads * d].reshape(n, heads, d)
    _check_attend(torch, pool, model, [n], qkv[:, :heads * d].reshape(n, heads, d), o, d ** -0.5, dtype, kv)


def test_rows_do_not_depend_on_the_batch(ta, gpu_ready):
    """A request's result bits with other requests beside it, twice, and on another stream: the same for the same hints."""
    torch = _t()
    rng = np.random.default_rng(41)
    kv, heads, d, dtype = 2, 4, 64, "bf16"
    lens = [900, 63, 128, 400]
    pool = _pool(ta, 4, 40, kv, d, "e4m3", dtype, 1024, 1600)
    model = ref.Model(4, kv, d, "e4m3", 40, 16)
    t = sum(lens) - 4
    _step(torch, pool, model, [n - 1 for n in lens], _tokens(rng, t, kv, d, dtype), _tokens(rng, t, kv, d, dtype), dtype)
    _step(torch, pool, model, [1] * 4, _tokens(rng, 4, kv, d, dtype), _tokens(rng, 4, kv, d, dtype), dtype)
    q = _dev(rng.standard_normal((4, heads, d)), dtype)
    outs = []
    side = torch.cuda.Stream()
    for s in (None, side, None):
        o = torch.empty_like(q)
        torch.cuda.synchronize()
        ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
        pool.attend(q, o, 0.125, max_new=1, max_len=900, workspace=ws, stream=s)
        torch.cuda.synchronize()
        outs.append(o)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_captured_steps(ta, gpu_ready):
    """A decode step (plan, append, attend) captured once and replayed with the pool's state advancing, eager work and
    a second captured step on another pool between the replays: every replay as the eager pool's step."""
    torch = _t()
    rng = np.random.default_rng(43)
    kv, heads, d, dtype, R = 2, 4, 64, "bf16", 3
    held = [62, 200, 5]

    def make():
        p = _pool(ta, R, 30, kv, d, "e4m3", dtype, 640, 300)
        m = ref.Model(R, kv, d, "e4m3", 30, 10)
        g = np.random.default_rng(1)
        t = sum(held)
        _step(torch, p, m, held, _tokens(g, t, kv, d, dtype), _tokens(g, t, kv, d, dtype), dtype)
        n = torch.ones(R, dtype=torch.int32, device="cuda")
        kvq = torch.zeros((R, (heads + 2 * kv) * d), dtype=torch.bfloat16, device="cuda")
        o = torch.zeros((R, heads * d), dtype=torch.bfloat16, device="cuda")
        ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")

        def step():
            p.step(n)
            p.append(kvq[:, heads * d:(heads + kv) * d], kvq[:, (heads + kv) * d:])
            p.attend(kvq[:, :heads * d], o, 0.125, max_new=1, max_len=640, workspace=ws)

        return p, kvq, o, step

    eager, e_in, e_out, e_step = make()
    graphs = []
    for _ in range(2):
        p, x, o, step = make()
        state = [t.clone() for t in (p.length, p.free_count, p.table)]
        g = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            step()
        for t, w in zip((p.length, p.free_count, p.table), state):
            assert torch.equal(t, w)  # captured, not run
        graphs.append((g, p, x, o, step))  # step holds the tensors that the graph reads
    for _ in range(6):
        x = _dev(rng.standard_normal(e_in.shape), dtype)
        e_in.copy_(x)
        e_step()
        torch.cuda.synchronize()
        for g, p, gx, go, _ in graphs:
            gx.copy_(x)
            go.fill_(-7)
            g.replay()
            torch.randn(1000, device="cuda").sum()
            torch.cuda.synchronize()
            assert torch.equal(go, e_out) and torch.equal(p.length, eager.length)
            assert torch.equal(p.slots, eager.slots) and torch.equal(p.status, eager.status)


def test_pool_keeps_its_workspace_on_other_streams(ta, gpu_ready, monkeypatch):
    """Split contexts without a caller's workspace: the pool's grows from call to call and from stream to stream, the
    memory that it lets go is not handed out while a call still uses it; a capture without one is refused."""
    torch = _t()
    rng = np.random.default_rng(53)
    kv, heads, d, dtype, n = 1, 4, 64, "bf16", 2000
    pool = _pool(ta, 1, 40, kv, d, "e4m3", dtype, 2560, 2000)
    model = ref.Model(1, kv, d, "e4m3", 40, 40)
    _step(torch, pool, model, [n], _tokens(rng, n, kv, d, dtype), _tokens(rng, n, kv, d, dtype), dtype)
    side = torch.cuda.Stream()
    for rows, stream in ((1, None), (4, side), (8, side.cuda_stream), (16, None), (24, side), (2, torch.cuda.default_stream())):
        q = _dev(rng.standard_normal((rows, heads, d)), dtype)
        pool.cu_tokens.copy_(torch.tensor([0, rows], dtype=torch.int32))
        hints = dict(max_new=rows, max_len=n)
        need = ta.kv8_attend_workspace(pool.cache, heads, rows, **hints)
        assert need > 0
        o, w = torch.empty_like(q), torch.empty_like(q)
        pool.attend(q, w, 0.125, workspace=torch.empty(need, dtype=torch.uint8, device="cuda"), **hints)
        torch.cuda.synchronize()
        pool.attend(q, o, 0.125, stream=stream, **hints)
        torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda")  # takes memory that is free
        torch.cuda.synchronize()
        assert torch.equal(o, w), rows
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ValueError):
        pool.attend(q, o, 0.125, **hints)


def test_pool_past_four_gigabytes(ta, gpu_ready):
    """Blocks whose bytes lie past 2^32 of K and V."""
    torch = _t()
    rng = np.random.default_rng(47)
    kv, heads, d, dtype, blocks = 8, 16, 128, "f16", 67000  # 4.39e9 bytes of K
    pool = ta.Kv8Pool(2, blocks, kv, d, max_len=512, max_tokens=400, dtype=torch.float16, code=ta.CODE_I8)
    model = ref.Model(2, kv, d, "i8", blocks, 8)
    pool.free_list.copy_(torch.arange(blocks, dtype=torch.int32))  # the last ids go first
    model.free = list(range(blocks))
    for n_new in ([130, 60], [1, 9]):
        t = sum(n_new)
        _step(torch, pool, model, n_new, _tokens(rng, t, kv, d, dtype), _tokens(rng, t, kv, d, dtype), dtype)
    assert pool.table[0, 0].item() * kv * 64 * d > 1 << 32
    q = _round(rng.standard_normal((10, heads, d)), dtype)
    o = torch.empty((10, heads, d), dtype=torch.float16, device="cuda")
    pool.attend(_dev(q, dtype), o, d ** -0.5)
    _check_attend(torch, pool, model, [1, 9], q, o, d ** -0.5, dtype, kv)
    t = pool.table[:, :2].flatten().long()
    t = t[t >= 0]
    got = pool.cache.k.view(torch.uint8)[t[0]].cpu().numpy()
    for h in range(kv):
        assert np.array_equal(got[h], model.block(0, 0, h, 0)[0])


# Steps whose rows per K/V head (new tokens times the heads that share it) pass 1024 go through another kernel.
MANY = [(code, dtype, d) for code in ("e4m3", "i8") for dtype in ("bf16", "f16") for d in (64, 128)]


@pytest.mark.parametrize("heads,kv,lens,news", [
    (24, 1, [130, 1, 64, 63], [130, 1, 60, 0]), (40, 2, [700, 64], [60, 64]), (21, 1, [3000], [50]),
    (3, 3, [1100, 129], [1090, 65]), (32, 1, [65, 190], [33, 2])])
@pytest.mark.parametrize("code,dtype,d", MANY)
def test_many_rows(ta, gpu_ready, code, dtype, d, heads, kv, lens, news):
    """Prompts, new tokens behind a cache, groups of heads that divide no tile, the keys split and not; scores that
    keep rising, so that the maximum moves; rows behind the last token stay."""
    torch = _t()
    rng = np.random.default_rng(sum(lens) + heads + d)
    total = sum(news)
    pool = _pool(ta, len(lens), sum(-(-n // 64) for n in lens), kv, d, code, dtype, 4096, sum(lens) + 3)
    model = ref.Model(len(lens), kv, d, code, pool.cache.blocks, 64)
    for n_new in ([n - m for n, m in zip(lens, news)], news):
        t = sum(n_new)
        k = _tokens(rng, t, kv, d, dtype) * np.linspace(0.2, 2.0, t)[:, None, None].astype(np.float32)
        _step(torch, pool, model, n_new, _round(k, dtype), _tokens(rng, t, kv, d, dtype, 30.0), dtype)
    q = _round(rng.standard_normal((total, heads, d)) * 2, dtype)
    qd = _dev(np.concatenate([q, np.zeros((3, heads, d), np.float32)]), dtype)
    for new, length in ((max(news), max(lens)), (0, 0), (max(news), 64)):
        o = torch.full_like(qd, -7.0)
        pool.attend(qd, o, d ** -0.5, max_new=new, max_len=length)
        assert (o[total:] == -7).all()
        _check_attend(torch, pool, model, news, q, o, d ** -0.5, dtype, kv)


@pytest.mark.parametrize("code,dtype,d", MANY)
def test_many_rows_no_numbers(ta, gpu_ready, code, dtype, d):
    """As for few rows: a NaN or infinity of a tail's V reaches the rows that read its token, of a block those that read
    the block, an infinite K of a masked token nothing, a table that names no block its own request."""
    torch = _t()
    rng = np.random.default_rng(d)
    heads, kv, held, news = 48, 2, 70, 50  # tokens 70 .. 119; the tail starts at 64; 1200 rows a K/V head
    n = held + news
    q = _round(rng.standard_normal((2 * news, heads, d)), dtype)
    keep = np.concatenate([np.arange(held), n + np.arange(held)])
    rest = np.concatenate([np.arange(held, n), n + np.arange(held, n)])
    k0, v0 = _tokens(rng, 2 * n, kv, d, dtype), _tokens(rng, 2 * n, kv, d, dtype)
    half = heads // kv
    for where, bad in (("v", float("nan")), ("v", float("inf")), ("k", -float("inf")), ("k_block", float("nan")),
                       ("v_block", float("inf")), ("table", 99), ("table", -1)):
        pool = _pool(ta, 2, 4, kv, d, code, dtype, 128, 2 * n)
        model = ref.Model(2, kv, d, code, 4, 2)
        k, v = k0.copy(), v0.copy()
        tok = 5 if "block" in where else 100  # of request 0, K/V head 1
        if where != "table":
            (k if where[0] == "k" else v)[tok, 1, 3] = bad
        _step(torch, pool, model, [held, held], k[keep], v[keep], dtype)
        _step(torch, pool, model, [news, news], k[rest], v[rest], dtype)
        if where == "table":
            pool.table[0, 0] = bad
        o = torch.empty((2 * news, heads, d), dtype=_dtype(dtype), device="cuda")
        pool.attend(_dev(q, dtype), o, d ** -0.5, max_new=news, max_len=n)
        isnan = torch.isnan(o).any(-1).cpu().numpy()
        want = np.zeros((2 * news, heads), bool)
        if where == "table":
            want[:news] = True
        elif "block" in where:
            want[:news, half:] = True
        else:
            want[tok - held:news, half:] = True
        if where == "v" and bad == bad:  # an infinity times a weight is one, or NaN where others meet it
            isnan |= torch.isinf(o).any(-1).cpu().numpy()
        if where == "k":  # rows that see it: a weight of 0 (a score of -inf) or NaN; the rows before are checked below
            isnan[tok - held:news, half:] = True
        assert np.array_equal(isnan, want), (where, bad)
        # the rows that do not see it are what they are without it
        if where in ("v", "k"):
            (model.v if where == "v" else model.k)[0][tok, 1, 3] = 0
            a, b, s = ref.attend(q[:tok - held, heads - 1], *model.values(0, 1), held + np.arange(tok - held), d ** -0.5)
            bound = ref.attend_bound(a, b, s, np.abs(model.values(0, 1)[1]).max(), n, HALF[dtype], dtype == "f16")
            assert (np.abs(o[:tok - held, heads - 1].float().cpu().numpy() - a) <= bound).all()
        _check_attend(torch, pool, model, [news, news], q, o, d ** -0.5, dtype, kv, skip=(0,))


@pytest.mark.parametrize("code,dtype,d,heads,kv", [("e4m3", "bf16", 64, 16, 16), ("i8", "f16", 64, 48, 4),
                                                   ("e4m3", "f16", 128, 48, 4), ("i8", "bf16", 128, 12, 12)])
@pytest.mark.parametrize("R", [13, 32])
def test_requests_taken_by_length(ta, gpu_ready, code, dtype, d, heads, kv, R):
    """Enough work that long requests go first: lengths that repeat, requests without tokens and new ones."""
    torch = _t()
    rng = np.random.default_rng(R + d + heads)
    held = [int(n) for n in rng.choice([0, 0, 1, 64, 130, 130, 250, 333], R)]
    news = [int(n) for n in rng.choice([0, 1, 7, 64, 70], R)] if R == 13 else [int(n) for n in rng.choice([0, 1, 9, 20], R)]
    news[3] = 100
    total = sum(news)
    pool = _pool(ta, R, sum(-(-(a + b) // 64) for a, b in zip(held, news)), kv, d, code, dtype, 512, sum(held) + total + 1)
    model = ref.Model(R, kv, d, code, pool.cache.blocks, 8)
    for n_new in (held, news):
        t = sum(n_new)
        _step(torch, pool, model, n_new, _tokens(rng, t, kv, d, dtype), _tokens(rng, t, kv, d, dtype), dtype)
    q = _round(rng.standard_normal((total, heads, d)), dtype)
    o = torch.empty((total, heads, d), dtype=_dtype(dtype), device="cuda")
    pool.attend(_dev(q, dtype), o, d ** -0.5, max_new=100, max_len=512)
    _check_attend(torch, pool, model, news, q, o, d ** -0.5, dtype, kv)


@pytest.mark.parametrize("d", [64, 128])
def test_captured_chunks(ta, gpu_ready, d):
    """A prompt's chunks (plan, append, attention of many rows) and the release of a request in one graph, replayed
    while the lengths advance: every replay as the eager pool's step."""
    torch = _t()
    rng = np.random.default_rng(67)
    kv, heads, dtype, R, n = 2, 36, "bf16", 2, 70

    def make():
        p = _pool(ta, R, 24, kv, d, "e4m3", dtype, 640, R * n)
        new = torch.tensor([n, n - 13], dtype=torch.int32, device="cuda")
        drop = torch.tensor([0, 1], dtype=torch.uint8, device="cuda")
        x = torch.zeros((R * n, (heads + 2 * kv) * d), dtype=torch.bfloat16, device="cuda")
        o = torch.zeros((R * n, heads * d), dtype=torch.bfloat16, device="cuda")
        ws = torch.empty(max(16, ta.kv8_attend_workspace(p.cache, heads, R * n, n, 640)), dtype=torch.uint8, device="cuda")

        def step():
            p.step(new)
            p.append(x[:, heads * d:(heads + kv) * d], x[:, (heads + kv) * d:])
            p.attend(x[:, :heads * d], o, d ** -0.5, max_new=n, max_len=640, workspace=ws)
            p.release(drop)

        return p, x, o, step

    eager, e_in, e_out, e_step = make()
    pool, g_in, g_out, step = make()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(5):
        x = _dev(rng.standard_normal(e_in.shape), dtype)
        e_in.copy_(x)
        g_in.copy_(x)
        g_out.fill_(-7)
        e_step()
        graph.replay()
        torch.randn(1000, device="cuda").sum()
        torch.cuda.synchronize()
        total = 2 * n - 13
        assert torch.equal(g_out[:total], e_out[:total]) and not torch.isnan(g_out[:total]).any()
        assert (g_out[total:] == -7).all()
        assert torch.equal(pool.length, eager.length) and pool.length[1].item() == 0
        assert torch.equal(pool.table, eager.table) and torch.equal(pool.free_count, eager.free_count)
    assert pool.length[0].item() == 5 * n


@pytest.mark.parametrize("d", [64, 128])
def test_many_rows_of_short_requests(ta, gpu_ready, d):
    """Counts that do not fit, with many rows: clamped as for few, the rows before a request's start 0."""
    torch = _t()
    rng = np.random.default_rng(d)
    heads, T = 24, 80
    pool = _pool(ta, 3, 12, 1, d, "e4m3", "bf16", 256, T)
    model = ref.Model(3, 1, d, "e4m3", 12, 4)
    k = _tokens(rng, T, 1, d, "bf16")
    _step(torch, pool, model, [40, 30, 10], k, k, "bf16")
    q, o = _dev(rng.standard_normal((T, heads, d)), "bf16"), torch.full((T, heads, d), -7.0, dtype=torch.bfloat16, device="cuda")
    big = (1 << 31) - 1
    for cu, length in (([0, 1000, 2000, big], [40, 30, 10]), ([-5, 90, 20, 10], [40, 30, 10]),
                       ([0, 40, 70, 80], [big, 30, 10]), ([0, 40, 70, 80], [-3, 30, 10])):
        pool.cu_tokens.copy_(torch.tensor(cu, dtype=torch.int32))
        pool.length.copy_(torch.tensor(length, dtype=torch.int32))
        pool.attend(q, o, 0.125, max_new=80)
    pool.cu_tokens.copy_(torch.tensor([0, 40, 70, 80], dtype=torch.int32))
    pool.length.copy_(torch.tensor([25, 30, 10], dtype=torch.int32))
    o.fill_(-7)
    pool.attend(q, o, 0.125, max_new=80)
    assert (o[:15] == 0).all() and (o[15:40] != 0).any()
    _check_attend(torch, pool, model, [40, 30, 10], q.float().cpu().numpy(), o, 0.125, "bf16", 1, skip=(0,))


def test_refusals_of_the_binding(ta, gpu_ready):
    """What the binding or the call refuses on real tensors: nothing is launched."""
    torch = _t()
    pool = _pool(ta, 2, 4, 2, 64, "e4m3", "bf16", 128, 16)
    pool.step(torch.tensor([3, 3], dtype=torch.int32, device="cuda"))
    x = torch.zeros((6, 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        pool.append(x.float(), x.float())
    with pytest.raises(ValueError):
        pool.append(x[:, :64], x[:, :64])
    with pytest.raises(ValueError):
        pool.attend(x, x[:3], 0.1)
    o = torch.empty_like(x)
    with pytest.raises(ta.TsfmError) as e:
        pool.attend(x, o, -1.0)
    assert e.value.code == ta.E_UNSUPPORTED
    with pytest.raises(ta.TsfmError) as e:  # three query heads for two of the cache
        pool.attend(torch.zeros((6, 192), dtype=torch.bfloat16, device="cuda"),
                    torch.zeros((6, 192), dtype=torch.bfloat16, device="cuda"), 0.1)
    assert e.value.code in (ta.E_INVALID, ta.E_UNSUPPORTED)
    wide = torch.zeros((6, 132), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ta.TsfmError) as e:  # a row stride of 264 bytes
        pool.append(wide[:, :128], wide[:, :128])
    assert e.value.code == ta.E_UNSUPPORTED
    big = _pool(ta, 1, 600, 1, 64, "e4m3", "bf16", 64 * 600, 1)
    q = torch.zeros((1, 64), dtype=torch.bfloat16, device="cuda")
    need = ta.kv8_attend_workspace(big.cache, 1, 1)
    assert need > 0
    rc = ta.kv8_attend(big.cache, q, q.clone(), big.cu_tokens, scale=0.1,
                       workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    assert rc == ta.E_INVALID and "workspace" in ta.last_error()
