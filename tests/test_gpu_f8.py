"""The e4m3 product with a scale per block of 128 (tsfm_f8_*) against float64: quantisation bit for bit, products with
bounds from the roundings that are made."""
import numpy as np
import pytest

import _kv8_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative


def _t():
    import torch

    return torch


def _dtype(name):
    return getattr(_t(), TYPES[name])


def _quantise_ref(x, group_rows):
    """codes and scales of f32-exact values, group by group: the scale from the finite values, NaN for the others."""
    rows, cols = x.shape
    codes = np.zeros((rows, cols), np.uint8)
    scales = np.zeros((-(-rows // group_rows), -(-cols // 128)), np.float32)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            g = np.s_[i * group_rows:(i + 1) * group_rows, j * 128:(j + 1) * 128]
            part = x[g].astype(np.float64)
            fin = np.abs(part[np.isfinite(part)])
            s = ref.e4m3_scale(fin.max() if fin.size else 0.0)
            scales[i, j] = s
            codes[g] = ref.e4m3_encode(part / s)
    return codes, scales


def _quantise(ta, x, group_rows, pad=0):
    torch = _t()
    rows, cols = x.shape
    codes = torch.full((rows, cols + pad), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((-(-rows // group_rows), -(-cols // 128)), -7.0, device="cuda")
    assert ta.f8_quantize(x, codes[:, :cols].view(torch.float8_e4m3fn), scales, group_rows) == ta.OK, ta.last_error()
    assert (codes[:, cols:] == 0x55).all()
    return codes, scales


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group_rows", [1, 128])
@pytest.mark.parametrize("rows,cols,pad", [(1, 16, 0), (3, 128, 16), (127, 144, 0), (129, 400, 32), (300, 1040, 0)])
def test_quantize_bit_for_bit(ta, gpu_ready, name, group_rows, rows, cols, pad):
    torch = _t()
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols)) * np.exp(3 * rng.standard_normal((rows, 1)))
    x = torch.from_numpy(x).to(_dtype(name)).cuda()
    codes, scales = _quantise(ta, x, group_rows, pad)
    want, s = _quantise_ref(x.float().cpu().numpy(), group_rows)
    assert np.array_equal(scales.cpu().numpy(), s)
    got = codes[:, :cols].cpu().numpy()
    assert np.array_equal(got, want)


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group_rows", [1, 128])
def test_quantize_extremes(ta, gpu_ready, name, group_rows):
    """Zeros, the smallest and largest values, both zeros' signs, midpoints between codes, 448 and just past it,
    values that are no numbers among them and alone."""
    torch = _t()
    fin = torch.finfo(_dtype(name))
    rows = [np.zeros(128), np.full(128, -fin.max), np.full(128, fin.tiny), np.full(128, fin.tiny / 2),
            np.tile([17.0, 19.0, -21.0, 0.0014648, 448.0, -0.0, 0.0, 2.0 ** -10], 16),
            np.tile([448.0, 1.0], 64), np.tile([450.0, 1.0], 64), np.tile([np.nan, 2.0, np.inf, -3.0], 32),
            np.full(128, np.nan), np.full(128, -np.inf)]
    x = np.zeros((len(rows) * 128 if group_rows == 128 else len(rows), 256))
    for i, r in enumerate(rows):
        x[i * group_rows, :128] = r
        x[i * group_rows, 128:] = r[::-1] * 0.5
    x = torch.from_numpy(x).to(_dtype(name)).cuda()
    codes, scales = _quantise(ta, x, group_rows)
    want, s = _quantise_ref(x.float().cpu().numpy(), group_rows)
    assert np.array_equal(scales.cpu().numpy(), s)
    got = codes.cpu().numpy()
    nan = (want & 127) == 127
    assert np.array_equal((got & 127) == 127, nan)  # a NaN's sign says nothing
    assert np.array_equal(got[~nan], want[~nan])


def _operands(rng, m, n, k, pad=0):
    torch = _t()
    kb, nb = -(-k // 128), -(-n // 128)

    def codes(rows):
        c = ref.e4m3_encode(np.clip(rng.standard_normal((rows, k)) * 60, -448, 448))
        full = np.full((rows, k + pad), 0x7f, np.uint8)  # NaN codes behind the rows: never read
        full[:, :k] = c
        return c, torch.from_numpy(full).cuda()[:, :k].view(torch.float8_e4m3fn)

    a, ad = codes(m)
    b, bd = codes(n)
    sa = np.exp(rng.standard_normal((m, kb))).astype(np.float32)
    sb = (rng.standard_normal((nb, kb)) * 0.01).astype(np.float32)  # of either sign
    return a, ad, sa, torch.from_numpy(sa).cuda(), b, bd, sb, torch.from_numpy(sb).cuda()


def _product_ref(a, sa, b, sb):
    """(c, S, M) in float64: the product, sum |a b|, and sum over blocks of 128 times the block's largest |a b|."""
    torch = _t()
    av, bv = (torch.from_numpy(ref.e4m3_decode(x)).cuda() for x in (a, b))
    m, k = av.shape
    n = bv.shape[0]
    c, S, M = (torch.zeros((m, n), dtype=torch.float64, device="cuda") for _ in range(3))
    for g in range(sa.shape[1]):
        x, y = av[:, g * 128:(g + 1) * 128], bv[:, g * 128:(g + 1) * 128]
        s = torch.from_numpy(sa[:, g].astype(np.float64)).cuda()[:, None] * \
            torch.from_numpy(np.repeat(sb[:, g], 128)[:n].astype(np.float64)).cuda()[None]
        c += s * (x @ y.t())
        S += s.abs() * (x.abs() @ y.abs().t())
        big = torch.zeros((m, n), dtype=torch.float64, device="cuda")
        for i in range(x.shape[1]):
            big = torch.maximum(big, x[:, i, None].abs() * y[None, :, i].abs())
        M += s.abs() * big * 128
    return c, S, M


def _bound(c, S, M, name, kbs):
    """The result's rounding; f32 sums: a partial sum of a block's 128 exact products and the sum over blocks, 2^-24 of
    at most S each; for 16-bit results the 8-bit instruction, which keeps the products of a step to about 2^-17 of the
    largest one (measured: an error of 2^-16 of a sum's norm over 128 normal values): 2^-17 for each of the 128."""
    b = HALF[name] * c.abs() + (130 + 2 * kbs) * 2.0 ** -24 * S + (2.0 ** -24 if name == "f16" else 0)
    return b if name == "f32" else b + 2.0 ** -17 * M


SHAPES = [(1, 16, 16), (1, 1, 128), (2, 130, 256), (15, 100, 112), (16, 64, 1040), (17, 129, 144), (33, 257, 384),
          (64, 1000, 128), (65, 48, 256), (100, 300, 400), (127, 127, 128), (129, 128, 272), (300, 520, 512),
          (513, 260, 640), (1030, 1100, 256)]


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_matches_float64(ta, gpu_ready, name, m, n, k):
    torch = _t()
    rng = np.random.default_rng(m * n + k)
    a, ad, sa, sad, b, bd, sb, sbd = _operands(rng, m, n, k, pad=16 if k % 128 else 0)
    wide = torch.full((m + 1, n + 3), -7.0, dtype=_dtype(name), device="cuda")
    assert ta.f8_gemm_nt(ad, sad, bd, sbd, wide[:m, :n]) == ta.OK, ta.last_error()
    assert (wide[m:] == -7).all() and (wide[:, n:] == -7).all()
    c, S, M = _product_ref(a, sa, b, sb)
    got = wide[:m, :n].double()
    bound = _bound(c, S, M, name, sa.shape[1])
    # a value past the type's largest (f16: 65504) has no finite rounding: infinity, of its sign, is the result
    past = torch.isinf(got) & (torch.sign(got) == torch.sign(c)) & (c.abs() + bound >= torch.finfo(_dtype(name)).max)
    err = torch.where(past, 0.0, (got - c).abs())
    assert (err <= bound).all(), float((err / bound).max())


# Few rows by 16, 32 and 64 columns a workgroup, tiles of 128 and of 256; reductions of 1 to 10 blocks.
WIDE = [(9, 4200, 144), (16, 8300, 272), (1, 16, 1280), (30, 4100, 256), (31, 8209, 144), (60, 4000, 1296),
        (130, 2100, 1152), (300, 2000, 1040), (20, 20000, 144), (1000, 2999, 656), (1100, 2900, 512), (2600, 1000, 896),
        (3500, 4200, 656), (3700, 4099, 128), (4000, 4096, 1040)]


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", WIDE)
def test_product_of_every_tile(ta, gpu_ready, name, m, n, k):
    """Each of the kernels, with rows of the result that start at 16 bytes and rows that do not: the same bits, within
    the bound, nothing written beside them."""
    torch = _t()
    rng = np.random.default_rng(m + n + k)
    a, ad, sa, sad, b, bd, sb, sbd = _operands(rng, m, n, k, pad=16)
    odd = torch.full((m + 1, n + 3 - n % 2), -7.0, dtype=_dtype(name), device="cuda")
    even = torch.full((m + 1, (n + 31) // 16 * 16), -7.0, dtype=_dtype(name), device="cuda")
    for wide in (odd, even):
        assert ta.f8_gemm_nt(ad, sad, bd, sbd, wide[:m, :n]) == ta.OK, ta.last_error()
        assert (wide[m:] == -7).all() and (wide[:, n:] == -7).all()
    assert torch.equal(odd[:m, :n], even[:m, :n])
    c, S, M = _product_ref(a, sa, b, sb)
    got = even[:m, :n].double()
    bound = _bound(c, S, M, name, sa.shape[1])
    ok = (got - c).abs() <= bound
    if name == "f16":  # a result that rounds past the largest value is an infinity
        ok |= got.isinf() & (c.abs() + bound >= torch.finfo(torch.float16).max)
    assert ok.all(), ((got - c).abs() / bound).max()


@pytest.mark.parametrize("m", [3, 70, 300])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_a_nan_stays_in_its_row_and_column(ta, gpu_ready, m, name):
    """A NaN code of a or b, or a NaN scale, makes exactly the outputs that read it NaN."""
    torch = _t()
    rng = np.random.default_rng(m)
    n, k = 200, 400
    a, ad, sa, sad, b, bd, sb, sbd = _operands(rng, m, n, k)
    ad.view(torch.uint8)[1, 390] = 0xff
    bd.view(torch.uint8)[7, 130] = 0x7f
    sad[2, 1] = float("nan")
    c = torch.empty((m, n), dtype=_dtype(name), device="cuda")
    assert ta.f8_gemm_nt(ad, sad, bd, sbd, c) == ta.OK
    want = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    want[1], want[2], want[:, 7] = True, True, True
    assert torch.equal(torch.isnan(c), want)
    sbd[1, 3] = float("nan")
    assert ta.f8_gemm_nt(ad, sad, bd, sbd, c) == ta.OK
    want[:, 128:] = True
    assert torch.equal(torch.isnan(c), want)


@pytest.mark.parametrize("m,n,k", [(1, 512, 512), (40, 300, 512), (700, 700, 512)])
def test_rows_do_not_depend_on_the_others(ta, gpu_ready, m, n, k):
    """Twice the same bits, and the same on another stream and in a captured graph."""
    torch = _t()
    rng = np.random.default_rng(m)
    _, ad, _, sad, _, bd, _, sbd = _operands(rng, m, n, k)
    outs = []
    side = torch.cuda.Stream()
    for s in (None, None, side):
        c = torch.empty((m, n), device="cuda")
        torch.cuda.synchronize()
        assert ta.f8_gemm_nt(ad, sad, bd, sbd, c, stream=s) == ta.OK
        torch.cuda.synchronize()
        outs.append(c)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    c, x = torch.empty((m, n), device="cuda"), torch.randn((m, k), device="cuda")
    codes = torch.empty((m, k), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((m, k // 128), device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert ta.f8_quantize(x, codes, scales) == ta.OK
        assert ta.f8_gemm_nt(codes, scales, bd, sbd, c) == ta.OK
    for i in range(4):
        x.normal_()
        c.fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        e = torch.empty_like(c)
        e_codes, e_scales = torch.empty_like(codes), torch.empty_like(scales)
        assert ta.f8_quantize(x, e_codes, e_scales) == ta.OK
        assert ta.f8_gemm_nt(e_codes, e_scales, bd, sbd, e) == ta.OK
        torch.cuda.synchronize()
        assert torch.equal(c, e), i


def test_nothing_to_do(ta, gpu_ready):
    torch = _t()
    e = torch.empty((0, 128), dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty((0, 1), device="cuda")
    b, sb = torch.empty((5, 128), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((1, 1), device="cuda")
    assert ta.f8_gemm_nt(e, s, b, sb, torch.empty((0, 5), device="cuda")) == ta.OK
    assert ta.f8_quantize(torch.empty((0, 128), device="cuda"), e, s) == ta.OK


def test_captured_products(ta, gpu_ready):
    """Quantisation and products of every kernel in one graph, replayed with other inputs and eager work between, and
    the same calls on a second stream at the same time: each result as the eager one."""
    torch = _t()
    rng = np.random.default_rng(61)
    shapes = [(1, 1000, 1024), (40, 500, 400), (300, 2000, 1040), (900, 1300, 640), (3500, 4200, 256)]
    calls = []
    for m, n, k in shapes:
        _, _, _, _, _, b, _, sb = _operands(rng, 1, n, k)
        calls.append((torch.empty((m, k), dtype=torch.bfloat16, device="cuda"), b, sb,
                      torch.empty((m, k), dtype=torch.float8_e4m3fn, device="cuda"),
                      torch.empty((m, -(-k // 128)), device="cuda"),
                      torch.empty((m, n), dtype=torch.bfloat16 if n % 1000 else torch.float32, device="cuda")))

    def run(outs, stream=None):
        for (x, b, sb, a, sa, _), c in zip(calls, outs):
            assert ta.f8_quantize(x, a, sa, stream=stream) == ta.OK
            assert ta.f8_gemm_nt(a, sa, b, sb, c, stream=stream) == ta.OK

    def fill():
        for x, *_ in calls:
            x.copy_(torch.randn(x.shape, device="cuda") * 3)

    fill()
    graph, outs = torch.cuda.CUDAGraph(), [c for *_, c in calls]
    with torch.cuda.graph(graph):
        run(outs)
    for _ in range(4):
        fill()
        for c in outs:
            c.fill_(-7)
        graph.replay()
        torch.randn(1000, device="cuda").sum()
        torch.cuda.synchronize()
        eager = [torch.empty_like(c) for c in outs]
        run(eager)
        for c, w in zip(outs, eager):
            assert torch.equal(c, w)
    # products of the same codes on two streams at once
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), [torch.empty_like(c) for c in outs]
    torch.cuda.synchronize()
    for _ in range(3):
        for (_, b, sb, a, sa, _), c, w in zip(calls, other, eager):
            assert ta.f8_gemm_nt(a, sa, b, sb, c, stream=side) == ta.OK
            assert ta.f8_gemm_nt(a, sa, b, sb, w) == ta.OK
    torch.cuda.synchronize()
    for c, o, w in zip(outs, other, eager):
        assert torch.equal(c, o) and torch.equal(c, w)


def test_serving_layer_in_8_bits(ta, gpu_ready):
    """The operators as a server runs them: two decode steps and a prompt through q/k/v in one 8-bit product, cache,
    attention and the output product, against the same in float64 from the GPU's own 8-bit activations (each product and
    the attention are checked for themselves elsewhere; here the way between them): relative error of the norm within the
    roundings that are made: bf16 q, k, v and o (2^-9 rms each at most), e4m3 K/V and e4m3 o (2^-5 rms at most each)."""
    torch = _t()
    rng = np.random.default_rng(3)
    R, heads, kv, d, model_d = 3, 8, 2, 64, 256
    width = (heads + 2 * kv) * d
    w = torch.randn((width, model_d), device="cuda") / 16
    w_o = torch.randn((model_d, heads * d), device="cuda") / 22

    def weights(x):
        c = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda")
        s = torch.empty((-(-x.shape[0] // 128), -(-x.shape[1] // 128)), device="cuda")
        assert ta.f8_quantize(x, c, s, group_rows=128) == ta.OK
        rows = s.repeat_interleave(128, 0)[:x.shape[0]].repeat_interleave(128, 1)[:, :x.shape[1]]
        return c, s, c.double() * rows.double()

    def linear(x, c, s, out):
        a = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device="cuda")
        sa = torch.empty((x.shape[0], -(-x.shape[1] // 128)), device="cuda")
        assert ta.f8_quantize(x, a, sa) == ta.OK
        y = torch.empty((x.shape[0], c.shape[0]), dtype=out, device="cuda")
        assert ta.f8_gemm_nt(a, sa, c, s, y) == ta.OK
        return y, a.double() * sa.double().repeat_interleave(128, 1)[:, :x.shape[1]]

    qkv_w, qkv_s, qkv_d = weights(w)
    o_w, o_s, o_d = weights(w_o)
    pool = ta.Kv8Pool(R, 16, kv, d, max_len=256, max_tokens=400)
    seen = [[torch.zeros((0, kv, d), dtype=torch.float64, device="cuda") for _ in range(2)] for _ in range(R)]
    for n_new in ([100, 7, 150], [1, 1, 1], [1, 0, 1]):
        t = sum(n_new)
        x = torch.randn((t, model_d), device="cuda")
        qkv, xd = linear(x, qkv_w, qkv_s, torch.bfloat16)
        pool.step(torch.tensor(n_new, dtype=torch.int32, device="cuda"))
        q, k, v = qkv[:, :heads * d], qkv[:, heads * d:(heads + kv) * d], qkv[:, (heads + kv) * d:]
        pool.append(k, v)
        o = torch.empty((t, heads * d), dtype=torch.bfloat16, device="cuda")
        pool.attend(q, o, d ** -0.5)
        y, _ = linear(o, o_w, o_s, torch.float32)
        assert pool.status.tolist()[0] == 0
        full = xd @ qkv_d.t()
        want, at = torch.zeros((t, heads * d), dtype=torch.float64, device="cuda"), 0
        for r, n in enumerate(n_new):
            rows = full[at:at + n]
            for i in range(2):
                part = rows[:, (heads + i * kv) * d:(heads + (i + 1) * kv) * d].reshape(n, kv, d)
                seen[r][i] = torch.cat([seen[r][i], part])
            kk, vv = seen[r]
            for h in range(heads):
                s = rows[:, h * d:(h + 1) * d] @ kk[:, h // (heads // kv)].t() * d ** -0.5
                last = len(kk) - n + torch.arange(n, device="cuda")[:, None]
                s = s.masked_fill(torch.arange(len(kk), device="cuda")[None] > last, -torch.inf)
                want[at:at + n, h * d:(h + 1) * d] = torch.softmax(s, -1) @ vv[:, h // (heads // kv)]
            at += n
        want = want @ o_d.t()
        rel = float((y.double() - want).norm() / want.norm())
        assert rel <= 3 * 2.0 ** -5 + 4 * 2.0 ** -9, rel
