"""Microscaled 4-bit floating point (rf_mxfp4.hip): codes and scales against the definition in 64 bits, bit
for bit; the product against the 64-bit product of the values they stand for; the 4-bit catalog's scores.

The product's tolerance: products of codes are exact, a sum of K terms in fp32 is within K u of the sum of
their sizes (u = 2^-24) in any order; the epilogue's two multiplications and one addition add 4 u of the
result's terms, the rounding to the output type eps / 2."""
import pytest
import torch

from recformer_amd import Mxfp4Catalog, ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def ref_quantize(x):
    """(codes (M, KB * 32) one a byte, scales (M, KB)) by the definition, in 64 bits on the CPU."""
    x = x.double().cpu()
    M, K = x.shape
    v = torch.nn.functional.pad(x, (0, -K % 32)).view(M, -1, 32)
    top = v.abs().amax(2)
    bad = ~torch.isfinite(v).all(2)
    top = torch.where(bad, torch.ones_like(top), top)
    e = torch.frexp(top).exponent - 1
    s = torch.where(top > 0, (e + 125).clamp(0, 254), torch.zeros_like(e))
    a = v.abs() * torch.pow(2.0, 127.0 - s.double())[:, :, None]
    d = (a[..., None] - GRID).abs()
    near = d == d.amin(-1, keepdim=True)  # one code, or two between which the even one is taken
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(near.sum(-1) > 1, even.int().argmax(-1), near.int().argmax(-1))
    code = torch.where(a > 6, torch.full_like(code, 7), code) | (torch.signbit(v).long() << 3)
    code[bad] = 0
    s[bad] = 255
    return code.view(M, -1), s


def codes_of(q):
    c = q.codes.cpu().long()
    return torch.stack([c & 15, c >> 4], 2).flatten(1)


def ref_values(q):
    """The 64-bit values of an Mxfp4 (device tensors), all blocks."""
    c = q.codes.long()
    c = torch.stack([c & 15, c >> 4], 2).flatten(1)
    v = GRID.to(c.device)[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    s = q.scales.double()
    f = torch.where(s == 255, torch.full_like(s, float("nan")), torch.pow(2.0, s - 127))
    return (v.view(c.shape[0], -1, 32) * f[:, :, None]).view(c.shape[0], -1)


def same_codes(q, x):
    code, s = ref_quantize(x)
    assert torch.equal(q.scales.cpu().long(), s)
    got = codes_of(q)
    zero = (code & 7) == 0  # the sign of a zero does not matter
    assert torch.equal(torch.where(zero & ((got & 7) == 0), code, got), code)


def rows_of(dev, dt, M, K, seed, layout="contiguous"):
    g = torch.Generator(device=dev).manual_seed(seed)
    v = torch.randn(M, K, device=dev, generator=g) * torch.exp2(torch.randint(-6, 7, (M, 1), device=dev, generator=g))
    v = v.to(dt)
    if layout == "contiguous":
        return v
    pad, off = (8, 0) if layout == "padded" else (3, 1)
    x = torch.full((M, K + pad), float("nan"), dtype=dt, device=dev)[:, off:off + K]
    x.copy_(v)
    return x


@pytest.mark.parametrize("layout", ["contiguous", "padded", "offset"])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 32), (3, 31), (5, 33), (70, 64), (9, 100), (130, 768), (2, 1000), (3, 4096)])
def test_quantise_and_back(dev, dt, M, K, layout):
    x = rows_of(dev, dt, M, K, M + K, layout)
    q, rn = ops.mxfp4_quantize(x, want_rnorm=True)
    assert q.codes.shape == (M, -(-K // 32) * 16) and q.scales.shape == (M, -(-K // 32)) and q.k == K
    same_codes(q, x)
    assert torch.equal(ops.mxfp4_quantize(x).codes, q.codes)
    want = ref_values(q)[:, :K]
    for out in DTYPES:
        got = ops.mxfp4_dequantize(q, out)
        assert got.dtype == out and torch.equal(got.double(), want.to(out).double())
    norm = 1.0 / x.double().square().sum(1).sqrt().clamp_min(1e-8)
    # the square sum's K roundings halve under the root, then a root and a division
    assert bool(((rn.double() - norm).abs() <= (K / 2 + 4) * U * norm).all())


@pytest.mark.parametrize("dt", DTYPES)
def test_every_rounding_border(dev, dt):
    """Each border between codes, its neighbours on both sides, both signs, beside 4 (which sets the scale to 1)
    and beside 7 (which saturates); exponents over the type's range; zeros; the smallest numbers."""
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
    eps = torch.finfo(dt).eps
    near = torch.cat([border, border * (1 + eps), border * (1 - eps)])
    vals = torch.cat([near, -near, torch.tensor([0.0, -0.0, 7.5, -7.5])]).to(dt)
    lo, hi = {torch.bfloat16: (-120, 120), torch.float16: (-10, 12), torch.float32: (-120, 120)}[dt]
    rows = []
    for e in (lo, -3, 0, 5, hi):
        for i in range(0, len(vals), 31):
            part = vals[i:i + 31].float()
            rows.append(torch.cat([torch.tensor([4.0]), part, torch.zeros(31 - len(part))]) * 2.0 ** e)
    tiny = torch.finfo(dt).smallest_normal
    for top in (tiny, tiny / 4, tiny * 8, torch.finfo(dt).max):
        rows.append(torch.linspace(-top, top, 32) if top < 1 else torch.linspace(-1, 1, 32) * top)
    rows.append(torch.zeros(32))
    x = torch.stack(rows).to(dt).to(dev)
    q = ops.mxfp4_quantize(x)
    same_codes(q, x)
    assert torch.equal(ops.mxfp4_dequantize(q).double(), ref_values(q).float().double())


@pytest.mark.parametrize("dt", DTYPES)
def test_nan_and_inf_make_their_block_nan(dev, dt):
    x = rows_of(dev, dt, 4, 96, 3)
    x[1, 40] = float("nan")
    x[2, 95] = float("inf")
    x[3, 0] = -float("inf")
    q = ops.mxfp4_quantize(x)
    same_codes(q, x)
    v = ops.mxfp4_dequantize(q)
    bad = torch.zeros(4, 3, dtype=torch.bool, device=dev)
    bad[1, 1] = bad[2, 2] = bad[3, 0] = True
    assert torch.equal(torch.isnan(v).view(4, 3, 32).all(2), bad) and torch.equal(torch.isnan(v).view(4, 3, 32).any(2), bad)
    w = ops.mxfp4_quantize(rows_of(dev, dt, 200, 96, 4))
    for rows in (4, 90):
        a = ops.Mxfp4(q.codes.repeat(-(-rows // 4), 1)[:rows].contiguous(),
                      q.scales.repeat(-(-rows // 4), 1)[:rows].contiguous(), 96)
        c = ops.mxfp4_gemm(a, w)
        want = bad.any(1).repeat(-(-rows // 4))[:rows]
        assert torch.equal(torch.isnan(c).all(1), want) and torch.equal(torch.isnan(c).any(1), want)


SHAPES = [(1, 1, 1), (1, 5, 32), (3, 70, 33), (16, 64, 768), (17, 129, 100), (33, 500, 160), (64, 1000, 768),
          (65, 127, 64), (128, 128, 128), (129, 257, 96), (200, 300, 1000), (300, 2000, 768), (1000, 130, 4096)]


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(dev, out, M, N, K):
    a = ops.mxfp4_quantize(rows_of(dev, torch.float32, M, K, 1))
    w = ops.mxfp4_quantize(rows_of(dev, torch.bfloat16, N, K, 2) * 0.1)
    va, vw = ref_values(a), ref_values(w)
    want, size = va @ vw.t(), va.abs() @ vw.abs().t()
    g = torch.Generator(device=dev).manual_seed(3)
    bias = torch.randn(N, device=dev, generator=g)
    ra, rw = torch.rand(M, device=dev, generator=g) + 0.5, torch.rand(N, device=dev, generator=g) + 0.5

    def close(got, ref, sz):
        lim = (K + 4) * U * sz + torch.finfo(out).eps / 2 * ref.abs() + torch.finfo(out).smallest_normal * 2 ** -10
        if out == torch.float16:
            ref = ref.clamp(-1e9, 1e9)
            over = ref.abs() + lim >= 65504
            got, ref, lim = got[~over], ref[~over], lim[~over]
        assert got.dtype == out
        d = (got.double() - ref).abs()
        assert bool((d <= lim).all()), float((d - lim).max())

    close(ops.mxfp4_gemm(a, w, out_dtype=out), want, size)
    close(ops.mxfp4_gemm(a, w, bias, out), want + bias.double(), size + bias.double().abs())
    f = ra.double()[:, None] * rw.double() * 0.05
    close(ops.mxfp4_gemm(a, w, None, out, ra, rw, 0.05), want * f, size * f)
    close(ops.mxfp4_gemm(a, w, bias, out, ra, rw, 0.05), want * f + bias.double(), size * f + bias.double().abs())


@pytest.mark.parametrize("M,N,K", [(2, 33000, 64), (5, 32769, 256), (16, 33001, 160), (16, 32770, 1600), (20, 20000, 96),
                                   (32, 33003, 128), (17, 40007, 33), (64, 32800, 512), (40, 33333, 200),
                                   (64, 33000, 1056), (33, 32768, 64), (50, 700, 1568)])
def test_product_of_few_rows_and_many_columns(dev, M, N, K):
    """Few rows against long tables, on both sides of where the work is laid out differently."""
    test_product(dev, torch.float32, M, N, K)


@pytest.mark.parametrize("M", [3, 100])
def test_scales_of_any_alignment(dev, M):
    """Tables of fewer than four scale bytes, and slices of a table, whose scales start anywhere."""
    for K in (20, 50, 96):
        test_product(dev, torch.float32, M, 1, K)
    w = ops.mxfp4_quantize(rows_of(dev, torch.bfloat16, 300, 224, 2))
    a = ops.mxfp4_quantize(rows_of(dev, torch.bfloat16, M + 5, 224, 3))
    whole = ops.mxfp4_gemm(a, w)
    for lo, hi in ((1, 300), (2, 131), (299, 300), (7, 140)):
        part = ops.Mxfp4(w.codes[lo:hi], w.scales[lo:hi], 224)
        assert torch.equal(ops.mxfp4_gemm(ops.Mxfp4(a.codes[5:], a.scales[5:], 224), part), whole[5:, lo:hi])
        assert torch.equal(ops.mxfp4_dequantize(part), ops.mxfp4_dequantize(w)[lo:hi])


def test_product_quantises_rows_on_the_way(dev):
    for dt in DTYPES:
        x = rows_of(dev, dt, 70, 200, 5, "offset")
        w = ops.mxfp4_quantize(rows_of(dev, dt, 90, 200, 6))
        got = ops.mxfp4_gemm(x, w)
        assert got.dtype == dt and torch.equal(got, ops.mxfp4_gemm(ops.mxfp4_quantize(x), w, out_dtype=dt))


def test_product_of_extreme_scales(dev):
    """Scale bytes 0 and 254 meet: 2^-127 times 2^127, exact; one row's scales do not touch another's."""
    for M in (3, 100):
        x = torch.zeros(M, 256, device=dev)
        x[:, :32] = 2.0 ** -125
        x[:, 200:] = 2.0 ** 100
        w = torch.zeros(70, 256, device=dev)
        w[:, :32] = 2.0 ** 126
        w[5, :32] = 0
        w[5, 200:] = 2.0 ** -100
        c = ops.mxfp4_gemm(x, ops.mxfp4_quantize(w))
        want = torch.full((M, 70), 64.0, device=dev)
        want[:, 5] = 56.0
        assert torch.equal(c, want)


def test_large_table_offsets(dev):
    """Rows behind 2^31 bytes of codes, in both kernels: a table of equal rows but the last ones."""
    N, K = 1100000, 4096
    codes = torch.full((N, K // 2), 0x22, dtype=torch.uint8, device=dev)  # all 1.0
    scales = torch.full((N, K // 32), 127, dtype=torch.uint8, device=dev)
    scales[-1] = 130
    w = ops.Mxfp4(codes, scales, K)
    for M in (2, 70):
        x = torch.ones(M, K, device=dev)
        c = ops.mxfp4_gemm(x, w)
        assert bool((c[:, :-1] == K).all()) and bool((c[:, -1] == 8 * K).all())
        del c


def test_catalog_scores_and_alternatives(dev):
    """The run they are made for: a 4-bit catalog's scores, a user's history masked, log probabilities with the
    best items, and a student taught by them."""
    from recformer_amd import train
    g = torch.Generator(device=dev).manual_seed(7)
    items = torch.randn(3001, 768, device=dev, generator=g).to(torch.bfloat16)
    users = torch.randn(70, 768, device=dev, generator=g).to(torch.bfloat16)
    cat = Mxfp4Catalog.from_items(items)
    assert cat.n == 3001
    s = cat.scores(users, temp=0.05)
    vu, vi = ref_values(ops.mxfp4_quantize(users)), ref_values(cat.table)
    f = 20.0 / users.double().norm(dim=1)[:, None] / items.double().norm(dim=1)
    want, size = (vu @ vi.t()) * f, (vu.abs() @ vi.abs().t()) * f
    assert bool(((s.double() - want).abs() <= (768 + 400) * U * size).all())  # norms: 768 / 2 + 4 each
    # four bits keep the scores near the cosines: each factor is off by at most 1/4 of a value
    true = (users.double() @ items.double().t()) * f
    assert float((s.double() - true).square().mean().sqrt()) < 0.25 * float(true.square().mean().sqrt())
    seen = torch.randint(0, 3001, (70, 20), device=dev, generator=g)
    s.scatter_(1, seen, -float("inf"))
    r = ops.token_logprobs(s, k=50, want_entropy=True)
    assert not bool((r.top_ids[:, :, None] == seen[:, None, :]).any())
    student = torch.randn(70, 3001, device=dev, generator=g).requires_grad_()
    loss = train.topk_distill_train(student, r.top_logp, r.top_ids)
    loss.backward()
    assert bool(torch.isfinite(student.grad).all()) and bool((student.grad.sum(1).abs() < 1e-6).all())


def test_replayed_and_side_by_side(dev):
    xs = [rows_of(dev, torch.bfloat16, 80, 768, s) for s in range(3)]
    w = ops.mxfp4_quantize(rows_of(dev, torch.bfloat16, 1000, 768, 9))
    cat = Mxfp4Catalog(w, torch.ones(1000, device=dev))

    def step(x):
        return [cat.scores(x, 0.05), cat.scores(x[:3], 0.05), ops.mxfp4_gemm(x, w)]

    eager = [step(x) for x in xs]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s, x in zip(side, xs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(step(x))
    torch.cuda.synchronize()
    for a, b in zip(eager, outs):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for k in (1, 2, 0, 1):
        static.copy_(xs[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, eager[k]))
        assert all(torch.equal(u, v) for u, v in zip(step(xs[2]), eager[2]))


def test_empty_and_refused(dev):
    w = ops.mxfp4_quantize(torch.ones(10, 64, device=dev))
    assert ops.mxfp4_quantize(torch.ones(0, 64, device=dev)).codes.shape == (0, 32)
    assert ops.mxfp4_gemm(torch.ones(0, 64, device=dev), w).shape == (0, 10)
    none = ops.mxfp4_quantize(torch.ones(0, 64, device=dev))
    assert ops.mxfp4_gemm(torch.ones(3, 64, device=dev), none).shape == (3, 0)
    x = torch.ones(3, 64, device=dev)
    with pytest.raises(ValueError):
        ops.mxfp4_gemm(torch.ones(3, 32, device=dev), w)
    with pytest.raises(ValueError):
        ops.mxfp4_gemm(x, w, torch.ones(9, device=dev))
    with pytest.raises(ValueError):
        ops.mxfp4_gemm(x, w, ra=torch.ones(3, device=dev))
    with pytest.raises(ValueError):
        ops.mxfp4_gemm(x, ops.Mxfp4(w.codes[:, :16], w.scales, 64))
    with pytest.raises(ValueError):
        ops.mxfp4_gemm(x, ops.Mxfp4(w.codes, w.scales.float(), 64))
    with pytest.raises(ValueError):
        ops.mxfp4_dequantize(ops.Mxfp4(w.codes, w.scales, 100))
    with pytest.raises(TypeError):
        ops.mxfp4_quantize(x.double())
    with pytest.raises(ValueError):
        ops.mxfp4_quantize(x.t())
    with pytest.raises(ValueError):
        ops.mxfp4_quantize(x[:1].expand(3, 64))
    with pytest.raises(ValueError):
        Mxfp4Catalog(w, torch.ones(9, device=dev))


@pytest.mark.parametrize("M,N", [(1, 40), (5, 33001), (64, 32900), (90, 70), (200, 300)])
def test_scale_without_row_and_column_factors(dev, M, N):
    """col_scale alone: a power of two is exact, with a bias the sum is rounded once more."""
    a = ops.mxfp4_quantize(rows_of(dev, torch.bfloat16, M, 96, 1))
    w = ops.mxfp4_quantize(rows_of(dev, torch.bfloat16, N, 96, 2))
    bias = torch.randn(N, device=dev)
    c = ops.mxfp4_gemm(a, w)
    assert torch.equal(ops.mxfp4_gemm(a, w, col_scale=0.25), c * 0.25)
    want = c.double() * 0.25 + bias.double()
    d = (ops.mxfp4_gemm(a, w, bias, col_scale=0.25).double() - want).abs()
    assert bool((d <= U * want.abs()).all())
    ones = torch.ones(max(M, N), device=dev)
    for out in DTYPES:  # factors of 1 change nothing
        assert torch.equal(ops.mxfp4_gemm(a, w, bias, out, col_scale=0.3),
                           ops.mxfp4_gemm(a, w, bias, out, ones[:M], ones[:N], 0.3))


def _at_any_byte(q):
    """q with its scales one byte off a word's border."""
    buf = torch.empty(q.scales.numel() + 8, dtype=torch.uint8, device=q.scales.device)
    s = buf[1:1 + q.scales.numel()].view(q.scales.shape)
    s.copy_(q.scales)
    return ops.Mxfp4(q.codes, s, q.k)


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("K", [96, 256, 512, 768, 800])
def test_product_of_several_tiles_a_workgroup(dev, out, K, aligned):
    """33 x 40 tiles, more than two for each workgroup there is, whole ones and those of an edge after one another,
    one to four steps of K each, different numbers in every row: the tile's limits as in test_product."""
    M, N = 4200, 5000
    a = ops.mxfp4_quantize(rows_of(dev, torch.float32, M, K, 1))
    w = ops.mxfp4_quantize(rows_of(dev, torch.bfloat16, N, K, 2) * 0.01)
    if not aligned:
        a, w = _at_any_byte(a), _at_any_byte(w)
    va, vw = ref_values(a), ref_values(w)
    want, size = va @ vw.t(), va.abs() @ vw.abs().t()
    g = torch.Generator(device=dev).manual_seed(3)
    bias = torch.randn(N, device=dev, generator=g)
    ra, rw = torch.rand(M, device=dev, generator=g) + 0.5, torch.rand(N, device=dev, generator=g) + 0.5

    def close(got, ref, sz):
        lim = (K + 4) * U * sz + torch.finfo(out).eps / 2 * ref.abs() + torch.finfo(out).smallest_normal * 2 ** -10
        keep = ref.abs() + lim < torch.finfo(out).max
        assert got.dtype == out
        d = (got.double() - ref).abs()
        assert bool((d <= lim)[keep].all()), float((d - lim)[keep].max())
        assert bool(keep.float().mean() > 0.99)

    close(ops.mxfp4_gemm(a, w, out_dtype=out), want, size)
    close(ops.mxfp4_gemm(a, w, bias, out), want + bias.double(), size + bias.double().abs())
    f = ra.double()[:, None] * rw.double() * 0.05
    close(ops.mxfp4_gemm(a, w, None, out, ra, rw, 0.05), want * f, size * f)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(2, 33000, 64), (5, 32769, 256), (16, 33001, 160), (16, 32770, 1600), (32, 33003, 128),
                                   (17, 40007, 33), (64, 32800, 512), (40, 50265, 768), (64, 33000, 1056)])
def test_product_of_few_rows_and_many_columns_in_16_bits(dev, out, M, N, K):
    test_product(dev, out, M, N, K)
