"""Log probabilities with entropy and alternatives, and distillation from a teacher's best logits
(rf_logprobs.hip): values and gradients against plain formulas in 64 bits, the order of the
alternatives against a stable sort, masks that leave a row empty, ties, NaN, strides and offsets, rows
of one column to a million, captured replays, refusals.

Tolerances, from the arithmetic (u = 2^-24, fp32's rounding): t = (x - m) it has two roundings, so
exp carries |t| 2u + 2u; a thread adds at most 64 values, the workgroup 6 + 16 partials and a join
some more, so s is within (100 + 2 |t|) u of its value with |t| averaged over the distribution (below
30 here): ln s is within 160 u absolute. logp: that plus 4u |logp|. The entropy divides two such sums:
2e-5 relative and absolute cover (180 + 160) u. Gradients: a rounding to the type (eps / 2), and 2e-5 of the
terms they are summed from; an exponential below 2^-126 is flushed to 0 (FLUSH, in units of the 2e-5)."""
import math

import pytest
import torch

from recformer_amd import ops, train

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
INF = float("inf")
U = 2.0 ** -24
FLUSH = 2.0 ** -126 / 2e-5
SIZES = [(1, 1), (2, 2), (3, 7), (700, 33), (5, 500), (9, 2049), (64, 10000), (3, 50265), (2, 65537), (2, 131075),
         (1, 1000003), (520, 4100)]


def logits_of(dev, dt, M, N, seed, layout="contiguous", scale=3.0):
    """(M, N) logits as a contiguous tensor, a view with padded rows, or one that starts off a 16-byte border."""
    g = torch.Generator(device=dev).manual_seed(seed)
    v = (torch.randn(M, N, device=dev, generator=g) * scale).to(dt)
    if layout == "contiguous":
        return v
    pad, off = (5, 0) if layout == "padded" else (3, 1)
    buf = torch.full((M, N + pad), float("nan"), dtype=dt, device=dev)
    x = buf[:, off:off + N]
    x.copy_(v)
    return x


def ref_softmax(x, it):
    """(logp, p, entropy) in 64 bits; -inf, 0, 0 for a row of nothing but -inf."""
    z = x.double()
    m = z.amax(1, keepdim=True)
    m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    e = ((z - m) * it).exp()
    s = e.sum(1, keepdim=True)
    logp = (z - m) * it - s.log()
    logp = torch.where(s == 0, torch.full_like(logp, -INF), logp)
    p = torch.where(s == 0, torch.zeros_like(e), e / s)
    return logp, p, -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)


def ref_grad(x, it, tokens, g, gh, ignore=-100):
    logp, p, h = ref_softmax(x, it)
    ok = tokens != ignore
    g = torch.where(ok, g.double(), torch.zeros_like(g.double()))
    w = torch.zeros_like(p).scatter_add_(1, tokens.clamp_min(0), g)
    lp = torch.where(p > 0, logp, torch.zeros_like(logp))
    d = it * (w - p * (g.sum(1, keepdim=True) + gh.double()[:, None] * (lp + h[:, None])))
    size = it * (w.abs() + (p + FLUSH) * (g.abs().sum(1, keepdim=True) + gh.double().abs()[:, None] * (lp.abs() + h[:, None])))
    empty = torch.isinf(x.double().amax(1)) & (x.double().amax(1) < 0)
    d[empty] = 0
    return d, size


def close_logp(got, want):
    # the answer is fp32: a log probability below its range (the lowest bf16 value times 20 is -6.8e39) rounds
    # to -inf, as this cast does, and any other moves by at most one of the 4 u
    want = want.float().double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isneginf(got), torch.isneginf(want))
    d = (got.double() - want)[fin].abs()
    assert bool((d <= 160 * U + 4 * U * want[fin].abs()).all()), float(d.max())


def close_grad(got, want, size):
    lim = torch.finfo(got.dtype).eps / 2 * want.abs() + 2e-5 * size + torch.finfo(got.dtype).smallest_normal * 2 ** -10
    d = (got.double() - want).abs()
    assert bool((d <= lim).all()), float((d - lim).max())


def check_top(x, r, k, it):
    ids = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.top_ids, ids)
    close_logp(r.top_logp, ref_softmax(x, it)[0].gather(1, ids))


@pytest.mark.parametrize("layout", ["contiguous", "padded", "offset"])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N", SIZES)
def test_logprobs_entropy_and_alternatives(dev, dt, M, N, layout):
    x = logits_of(dev, dt, M, N, M + N, layout)
    g = torch.Generator(device=dev).manual_seed(N)
    tokens = torch.randint(0, N, (M, 3), device=dev, generator=g)
    tokens[0, 1] = -100
    k = min(N, 20)
    r = ops.token_logprobs(x, tokens, k=k, inv_temp=0.7, want_entropy=True)
    logp, _, h = ref_softmax(x, 0.7)
    want = torch.where(tokens == -100, torch.zeros_like(logp[:, :1]), logp.gather(1, tokens.clamp_min(0)))
    close_logp(r.logp, want)
    assert bool(((r.entropy.double() - h).abs() <= 2e-5 + 2e-5 * h).all())
    check_top(x, r, k, 0.7)
    one = ops.token_logprobs(x, tokens[:, 0].to(torch.int32), inv_temp=0.7)  # (M,) and int32 ids
    assert one.logp.shape == (M,) and one.entropy is None and one.top_ids is None
    close_logp(one.logp, want[:, 0])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,k", [(3, 3), (300, 256), (2500, 256), (5000, 1), (30000, 64), (30000, 65), (30000, 256),
                                 (200000, 256)])
def test_alternatives_of_every_length(dev, dt, N, k):
    for M in (1, 6):
        x = logits_of(dev, dt, M, N, N + k)
        check_top(x, ops.token_logprobs(x, k=k), k, 1.0)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N", [(4, 700), (4, 9000), (2, 70000), (1, 400000)])
def test_alternatives_with_ties(dev, dt, M, N):
    """Equal logits go by index: few values, one value, all the best in one 16-byte chunk or in neighbours."""
    g = torch.Generator(device=dev).manual_seed(N)
    few = torch.randint(-2, 3, (M, N), device=dev, generator=g).to(dt)
    check_top(few, ops.token_logprobs(few, k=100), 100, 1.0)
    same = torch.full((M, N), -1.5, device=dev, dtype=dt)
    check_top(same, ops.token_logprobs(same, k=256), 256, 1.0)
    run = logits_of(dev, dt, M, N, 3)
    run[:, N // 2:N // 2 + 400] = 50.0
    check_top(run, ops.token_logprobs(run, k=256), 256, 1.0)
    up = torch.arange(N, device=dev).float().div(N).expand(M, N).to(dt).contiguous()
    check_top(up, ops.token_logprobs(up, k=50), 50, 1.0)
    zeros = torch.zeros(M, N, device=dev, dtype=dt)
    zeros[:, ::2] = -0.0
    check_top(zeros, ops.token_logprobs(zeros, k=8), 8, 1.0)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N", [5, 900, 20000, 140000])
def test_masked_rows(dev, dt, N):
    """-inf columns, rows of nothing else, rows with one column left, rows of the type's lowest value, and
    a mask of the lowest value beside ordinary logits: values, alternatives and gradients."""
    x = logits_of(dev, dt, 6, N, N)
    low = torch.finfo(dt).min
    x[0] = -INF
    x[1] = -INF
    x[1, N - 1] = 2.0
    x[2] = low
    x[3, ::2] = -INF
    x[4, 1:] = low
    tokens = torch.tensor([[0, N - 1]] * 6, device=dev)
    it = 20.0 if dt != torch.float32 else 1.0
    r = ops.token_logprobs(x, tokens, k=min(N, 5), inv_temp=it, want_entropy=True, want_stats=True)
    logp, p, h = ref_softmax(x, it)
    close_logp(r.logp, logp.gather(1, tokens))
    assert bool(((r.entropy.double() - h).abs() <= 2e-5 + 2e-5 * h).all())
    ids = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :min(N, 5)]
    assert torch.equal(r.top_ids, ids)
    g = torch.tensor([[1.0, -0.5]] * 6, device=dev)
    gh = torch.full((6,), 0.25, device=dev)
    d = ops.token_logprobs_bwd(x, r.stats, tokens, g, r.entropy, gh, it)
    want, size = ref_grad(x, it, tokens, g, gh)
    close_grad(d, want, size)
    assert not bool(d[0].any())


@pytest.mark.parametrize("N", [40, 5000, 100000])
def test_nan_and_inf_rows(dev, N):
    x = logits_of(dev, torch.float32, 4, N, 1)
    clean = x.clone()
    x[1, N // 2] = float("nan")
    x[2, N // 3] = INF
    r = ops.token_logprobs(x, torch.zeros(4, dtype=torch.long, device=dev), k=4, want_entropy=True)
    c = ops.token_logprobs(clean, torch.zeros(4, dtype=torch.long, device=dev), k=4, want_entropy=True)
    for a, b in ((r.logp, c.logp), (r.entropy, c.entropy), (r.top_logp, c.top_logp)):
        assert bool(torch.isnan(a[1:3]).all())
        assert torch.equal(a[[0, 3]], b[[0, 3]])
    assert torch.equal(r.top_ids[[0, 3]], c.top_ids[[0, 3]])
    assert r.top_ids[1, 0] == N // 2 and r.top_ids[2, 0] == N // 3  # still the order of the logits
    assert torch.equal(r.top_ids[2, 1:], clean[2].masked_fill(torch.arange(N, device=dev) == N // 3, -INF)
                       .sort(descending=True, stable=True).indices[:3])


def test_ids_out_of_range(dev):
    x = logits_of(dev, torch.float32, 4, 100, 2)
    tokens = torch.tensor([5, 100, -7, -100], device=dev)
    r = ops.token_logprobs(x, tokens, want_stats=True)
    assert bool(torch.isfinite(r.logp[0])) and bool(torch.isnan(r.logp[1:3]).all()) and r.logp[3] == 0
    d = ops.token_logprobs_bwd(x, r.stats, tokens, torch.ones(4, device=dev))
    assert bool(torch.isfinite(d[0]).all()) and bool(torch.isnan(d[1:3]).all()) and not bool(d[3].any())
    r = ops.token_logprobs(x, tokens, ignore_index=5)
    assert r.logp[0] == 0 and bool(torch.isnan(r.logp[3]))
    ids = torch.tensor([[1, 2], [1, 100], [-2, 3], [-1, -1]], device=dev)
    rows, stats, loss, coef = ops.topk_distill(x, torch.zeros(4, 2, device=dev), ids)
    assert bool(torch.isfinite(rows[0])) and bool(torch.isnan(rows[1:3]).all()) and rows[3] == 0
    d = ops.topk_distill_bwd(x, stats, torch.zeros(4, 2, device=dev), ids, torch.ones(1, device=dev), coef)
    assert bool(torch.isfinite(d[0]).all()) and bool(torch.isnan(d[1:3]).all()) and not bool(d[3].any())


@pytest.mark.parametrize("layout", ["contiguous", "padded", "offset"])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N", SIZES)
def test_logprobs_gradient(dev, dt, M, N, layout):
    x = logits_of(dev, dt, M, N, 7 * M + N, layout)
    g = torch.Generator(device=dev).manual_seed(N)
    tokens = torch.randint(0, N, (M, 4), device=dev, generator=g)
    tokens[:, 3] = tokens[:, 0]  # the same entry twice
    tokens[0, 2] = -100
    w = torch.randn(M, 4, device=dev, generator=g)
    wh = torch.randn(M, device=dev, generator=g)
    leaf = x.detach().requires_grad_()
    logp, h = train.token_logprobs_train(leaf, tokens, inv_temp=1.3)
    both, = torch.autograd.grad((logp, h), leaf, (w, wh), retain_graph=True)
    want, size = ref_grad(x, 1.3, tokens, w, wh)
    assert both.dtype == dt and both.shape == x.shape
    close_grad(both, want, size)
    only, = torch.autograd.grad(logp, leaf, w, retain_graph=True)
    close_grad(only, *ref_grad(x, 1.3, tokens, w, torch.zeros_like(wh)))
    only, = torch.autograd.grad(h.sum(), leaf)  # an expanded upstream gradient
    close_grad(only, *ref_grad(x, 1.3, tokens, torch.zeros_like(w), torch.ones_like(wh)))


def ref_distill(x, tl, ids, temp):
    """(rows, gradient of their sum, size of its terms) in 64 bits; temp^2 left out."""
    it = 1.0 / temp
    logp, p, _ = ref_softmax(x, it)
    q = ref_softmax(torch.where(ids >= 0, tl.double(), torch.full_like(tl.double(), -INF)), it)[1]
    at = ids.clamp_min(0)
    lq = torch.where(q > 0, q.log(), torch.zeros_like(q))
    rows = torch.where(q > 0, q * (lq - logp.gather(1, at)), torch.zeros_like(q)).sum(1)
    used = q.sum(1, keepdim=True)
    taught = torch.zeros_like(p).scatter_add_(1, at, q)
    return rows, it * (p * used - taught), it * ((p + FLUSH) * used + taught), used[:, 0] > 0


@pytest.mark.parametrize("layout", ["contiguous", "padded", "offset"])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N", SIZES)
def test_distillation(dev, dt, M, N, layout):
    x = logits_of(dev, dt, M, N, 11 * M + N, layout)
    g = torch.Generator(device=dev).manual_seed(N)
    for K in sorted({1, min(N, 5), 64, 300}):
        ids = torch.randint(0, N, (M, K), device=dev, generator=g)  # repeated ids where N is small
        tl = torch.randn(M, K, device=dev, generator=g) * 2
        ids[torch.rand(M, K, device=dev, generator=g) < 0.2] = -1
        if K > 1:
            tl[0, 0] = -INF
        if M > 2:
            ids[1] = -1
        if not bool((ids[0] >= 0).any()):
            ids[0, K - 1] = 0
        leaf = x.detach().requires_grad_()
        loss = train.topk_distill_train(leaf, tl, ids, temp=1.7)
        d, = torch.autograd.grad(loss * 3.0, leaf)
        rows, dr, size, used = ref_distill(x, tl, ids, 1.7)
        n = int(used.sum())
        got, stats, mean, coef = ops.topk_distill(x, tl, ids, 1.0 / 1.7, 2.0)
        lim = 2e-5 * (1.0 + rows.abs() + 2 * math.log(N + 1) + 10)  # ln q, ln p and their weighted sums
        assert bool(((got.double() - rows).abs() <= lim).all())
        assert torch.equal(stats[:, 3] > 0, used)
        f = 1.7 ** 2 / n
        assert abs(float(loss.detach()) - float(rows.sum()) * f) <= f * float(lim.sum())
        assert abs(float(mean) - float(rows.sum()) * 2 / n) <= 2 / n * float(lim.sum())
        assert abs(float(coef) - 2 / n) <= 4 * U * 2 / n
        close_grad(d, dr * (3 * f), size * (3 * f))


def test_distillation_of_masked_rows(dev):
    """A taught column that the student masks: an infinite loss, the formula's gradient elsewhere; a student
    row of nothing: gradient 0; no row that lists anything: nan, as a mean cross entropy over no row."""
    x = logits_of(dev, torch.float32, 3, 50, 5)
    x[0, 7] = -INF
    x[1] = -INF
    ids = torch.tensor([[7, 8], [1, 2], [3, 4]], device=dev)
    tl = torch.tensor([[0.0, 1.0]] * 3, device=dev)
    rows, stats, _, coef = ops.topk_distill(x, tl, ids)
    assert torch.isposinf(rows[0]) and torch.isposinf(rows[1]) and bool(torch.isfinite(rows[2]))
    d = ops.topk_distill_bwd(x, stats, tl, ids, torch.ones((), device=dev), torch.ones((), device=dev))
    _, want, size, _ = ref_distill(x, tl, ids, 1.0)
    close_grad(d[[0, 2]], want[[0, 2]], size[[0, 2]])
    assert not bool(d[1].any())
    leaf = x.detach().requires_grad_()
    assert torch.isnan(train.topk_distill_train(leaf, tl, torch.full_like(ids, -1)))


@pytest.mark.parametrize("N", [77, 50265])
def test_gradients_against_differences(dev, N):
    """Central differences of the fp32 kernels' own forward along a random direction. A step of 0.05 leaves
    third-order terms below 0.05^2 / 6 of a bounded third derivative (< 1 for sums of these weights) and a
    rounding noise of 2 * 2e-5 * 20 / 0.1 in the quotient."""
    g = torch.Generator(device=dev).manual_seed(N)
    x = logits_of(dev, torch.float32, 2, N, N)
    v = torch.randn(2, N, device=dev, generator=g)
    v = v / v.abs().max()
    tokens = torch.tensor([[1], [N - 1]], device=dev)
    ids = torch.tensor([[0, 5, 9], [2, 5, 70]], device=dev)
    tl = torch.randn(2, 3, device=dev, generator=g)

    def f(y):
        logp, h = train.token_logprobs_train(y, tokens)
        return logp.sum() + 0.5 * h.sum() + train.topk_distill_train(y, tl, ids, 2.0)

    leaf = x.clone().requires_grad_()
    grad, = torch.autograd.grad(f(leaf), leaf)
    want = float(f(x + 0.05 * v).double() - f(x - 0.05 * v).double()) / 0.1
    got = float((grad.double() * v.double()).sum())
    assert abs(got - want) <= 0.05 ** 2 + 2 * 2e-5 * 20 / 0.1, (got, want)


def test_rows_stay_within_their_bounds(dev):
    """The gradient of a view writes its own columns only, and rows behind the last stay as they were."""
    buf = torch.full((6, 40), 9.0, device=dev)
    x = buf[1:4, 5:33]
    x.copy_(logits_of(dev, torch.float32, 3, 28, 1))
    r = ops.token_logprobs(x, torch.zeros(3, dtype=torch.long, device=dev), k=3, want_stats=True)
    d = ops.token_logprobs_bwd(x, r.stats, torch.zeros(3, dtype=torch.long, device=dev), torch.ones(3, device=dev))
    assert d.stride(1) == 1 and d.data_ptr() % 16 == x.data_ptr() % 16
    keep = buf.clone()
    keep[1:4, 5:33] = 9.0
    assert bool((keep == 9.0).all())
    empty = ops.token_logprobs(x[:0], torch.zeros(0, dtype=torch.long, device=dev), k=2, want_entropy=True)
    assert empty.logp.shape == (0,) and empty.top_ids.shape == (0, 2) and empty.entropy.shape == (0,)
    none = ops.token_logprobs(x, torch.zeros(3, 0, dtype=torch.long, device=dev), k=1)
    assert none.logp.shape == (3, 0) and none.top_ids.shape == (3, 1)


@pytest.mark.parametrize("M,N", [(1, 50265), (40, 10000)])
def test_same_results_alone_side_by_side_and_replayed(dev, M, N):
    """Bit-identical from call to call, on two streams at once, and in a captured graph replayed on new inputs
    between eager calls."""
    xs = [logits_of(dev, torch.bfloat16, M, N, s) for s in range(3)]
    tokens = torch.arange(M, device=dev)
    tl = torch.randn(M, 8, device=dev)
    ids = torch.randint(0, N, (M, 8), device=dev)

    def step(x):
        leaf = x.detach().requires_grad_()
        logp, h = train.token_logprobs_train(leaf, tokens)
        loss = train.topk_distill_train(leaf, tl, ids, 2.0)
        d, = torch.autograd.grad(loss + logp.sum() + h.sum(), leaf)
        r = ops.token_logprobs(x, tokens, k=9, want_entropy=True)
        return [logp.detach(), h.detach(), loss.detach(), d, r.top_logp, r.top_ids]

    eager = [step(x) for x in xs]
    again = [step(x) for x in xs]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s, x in zip(side, xs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(step(x))
    torch.cuda.synchronize()
    for a, b in list(zip(eager, again)) + list(zip(eager, outs)):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    static = xs[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(static)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for k in (1, 2, 0, 1):
        static.copy_(xs[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, eager[k]))
        assert all(torch.equal(u, v) for u, v in zip(step(xs[2]), eager[2]))


def test_teacher_alternatives_into_distillation(dev):
    """The run they are made for: a teacher's alternatives and their log probabilities, a student taught by
    them; a student equal to the teacher on the listed entries' softmax has the smallest loss there is."""
    teacher = logits_of(dev, torch.bfloat16, 8, 5000, 3)
    r = ops.token_logprobs(teacher, k=50)
    leaf = logits_of(dev, torch.bfloat16, 8, 5000, 4).requires_grad_()
    loss = train.topk_distill_train(leaf, r.top_logp, r.top_ids, temp=1.0)
    d, = torch.autograd.grad(loss, leaf)
    rows, want, size, _ = ref_distill(leaf.detach(), r.top_logp, r.top_ids, 1.0)
    assert abs(float(loss.detach()) - float(rows.mean())) <= 2e-5 * 40
    close_grad(d, want / 8, size / 8)
    listed = torch.full((8, 5000), -INF, device=dev).scatter(1, r.top_ids, r.top_logp)
    rows, *_ = ops.topk_distill(listed, r.top_logp, r.top_ids)
    assert bool((rows.abs() <= 2e-5 * 40).all())


def test_refusals(dev):
    x = torch.zeros(4, 50, device=dev)
    tok = torch.zeros(4, dtype=torch.long, device=dev)
    for bad in (0.0, -1.0, float("nan"), INF):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, tok, inv_temp=bad)
    for k in (-1, 51, 257):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, tok, k=k)
    with pytest.raises(ValueError):
        ops.token_logprobs(x)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, tok[:3])
    with pytest.raises(TypeError):
        ops.token_logprobs(x, tok.float())
    with pytest.raises(ValueError):
        ops.token_logprobs(x, tok.cpu())
    with pytest.raises(TypeError):
        ops.token_logprobs(x.double(), tok)
    with pytest.raises(ValueError):
        ops.token_logprobs(x.t(), torch.zeros(50, dtype=torch.long, device=dev))
    with pytest.raises(ValueError):
        ops.token_logprobs(x[:1].expand(4, 50), tok)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, torch.zeros(4, 1025, dtype=torch.long, device=dev))
    with pytest.raises(ValueError):
        ops.topk_distill(x, torch.zeros(4, 3, device=dev), torch.zeros(4, 2, dtype=torch.long, device=dev))
    with pytest.raises(ValueError):
        ops.topk_distill(x, torch.zeros(4, 0, device=dev), torch.zeros(4, 0, dtype=torch.long, device=dev))
    with pytest.raises(ValueError):
        train.topk_distill_train(x, torch.zeros(4, 2, device=dev), torch.zeros(4, 2, dtype=torch.long, device=dev), 0.0)
    with pytest.raises(ValueError):
        ops.token_logprobs_bwd(x, torch.zeros(4, 3, device=dev), tok, torch.ones(4, device=dev))


def test_model_answers_and_learns_from_a_teacher(dev):
    """RecformerForSeqRec.item_logprobs / distill_loss and RecformerForPretraining.token_logprobs: the numbers of
    the scores they come from, a history left out, and parameter gradients equal to autograd's through the
    plain formula on the same scores (the backward below the scores is the same: 1e-5 of the largest, from
    the 2e-5 of the scores' gradients)."""
    from recformer_amd.hashinit import hash_tensor
    from recformer_amd.models import RecformerForSeqRec
    from recformer_amd.synth import C1, synth_batch
    from tests.common import hashed_model, hashed_pretrain
    m = hashed_model(dict(C1, item_num=300), 1, RecformerForSeqRec)
    m.init_item_embedding(hash_tensor("items", (300, C1["hidden_size"]), "weight", std=1.0))
    m = m.to(dev)
    batch = {k: v.to(dev) for k, v in synth_batch(4, 96, C1["vocab_size"], seed=1).items()}
    with torch.no_grad():
        z = m.longformer(**batch).pooler_output
        scores = m.similarity_score(z)
    seen = torch.tensor([[3, 5], [0, -1], [-1, -1], [7, 7]], device=dev)
    r = m.item_logprobs(z, torch.tensor([3, 1, 2, 9], device=dev), k=10, seen=seen, want_entropy=True)
    masked = scores.clone()
    masked[0, [3, 5]] = -INF
    masked[1, 0] = -INF
    masked[3, 7] = -INF
    logp, _, h = ref_softmax(masked, 1.0)
    close_logp(r.logp, logp[torch.arange(4), [3, 1, 2, 9]])
    check_top(masked, r, 10, 1.0)
    teacher = ops.token_logprobs(torch.randn(4, 300, device=dev), k=20)
    loss = m.distill_loss(teacher.top_logp, teacher.top_ids, 2.0, **batch)
    loss.backward()
    got = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}
    assert got
    m.zero_grad(set_to_none=True)
    s = m(**batch)
    ls = torch.log_softmax(s.double() / 2.0, 1)
    lq = torch.log_softmax(teacher.top_logp.double() / 2.0, 1)
    plain = 4.0 * (lq.exp() * (lq - ls.gather(1, teacher.top_ids))).sum(1).mean()
    assert abs(float(plain.detach()) - float(loss.detach())) <= 4.0 * 2e-5 * 40
    plain.backward()
    for n, g in got.items():
        w = dict(m.named_parameters())[n].grad
        assert float((g - w).abs().max()) <= 1e-3 * float(w.abs().max()) + 1e-9, n
    lm = hashed_pretrain(C1).to(dev)
    hidden = torch.randn(5, C1["hidden_size"], device=dev)
    words = torch.tensor([1, 2, -100, 4, 5], device=dev)
    r = lm.token_logprobs(hidden, words, k=3)
    logits = lm.lm_logits(hidden)
    close_logp(r.logp, torch.where(words < 0, 0.0, ref_softmax(logits, 1.0)[0].gather(1, words.clamp_min(0)[:, None])[:, 0]))
    check_top(logits, r, 3, 1.0)


@pytest.mark.parametrize("N,pad", [(50, 6), (4100, 3)])
def test_gradients_through_saved_tensor_hooks(dev, N, pad):
    """Hooks that keep saved tensors elsewhere (offloading) may hand the logits back with other strides: the
    gradient is the same."""
    buf = torch.full((5, N + pad), float("nan"), device=dev)
    buf[:, :N] = logits_of(dev, torch.float32, 5, N, 3)
    ids = torch.randint(0, N, (5, 4), device=dev)
    tl = torch.randn(5, 4, device=dev)

    def grads(x):
        leaf = x.detach().requires_grad_()
        logp, h = train.token_logprobs_train(leaf, ids)
        loss = train.topk_distill_train(leaf, tl, ids, 2.0)
        return leaf, loss + logp.sum() + h.sum()

    leaf, out = grads(buf[:, :N])
    want, = torch.autograd.grad(out, leaf)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t):
        leaf, out = grads(buf[:, :N])
    got, = torch.autograd.grad(out, leaf)
    assert torch.equal(got, want)


def test_second_derivatives_are_refused(dev):
    ids = torch.tensor([[1, 2], [3, 4]], device=dev)
    for fn in (lambda x: train.token_logprobs_train(x, ids)[0].sum(),
               lambda x: train.token_logprobs_train(x, ids)[1].sum(),
               lambda x: train.topk_distill_train(x, torch.randn(2, 2, device=dev), ids)):
        leaf = logits_of(dev, torch.float32, 2, 50, 1).requires_grad_()
        d, = torch.autograd.grad(fn(leaf), leaf, create_graph=True)
        assert bool(torch.isfinite(d).all())
        with pytest.raises(RuntimeError):
            d.square().sum().backward()


def test_history_ids_outside_the_catalog_leave_out_nothing(dev):
    """A padding id of N, or an id of another catalog, in the history; int32 ids; no slot at all; a history of
    other users; and batches that would not give the catalog's scores are refused."""
    from recformer_amd.hashinit import hash_tensor
    from recformer_amd.models import RecformerForSeqRec
    from recformer_amd.synth import C1
    from tests.common import hashed_model
    m = hashed_model(dict(C1, item_num=70), 1, RecformerForSeqRec)
    m.init_item_embedding(hash_tensor("items", (70, C1["hidden_size"]), "weight", std=1.0))
    m = m.to(dev)
    z = torch.randn(2, C1["hidden_size"], device=dev)
    want = m.item_logprobs(z, k=70, seen=torch.tensor([[69, 4], [0, -1]], device=dev))
    got = m.item_logprobs(z, k=70, seen=torch.tensor([[69, 4, 70, 2 ** 30], [70, 0, -5, 71]], device=dev, dtype=torch.int32))
    assert torch.equal(want.top_ids, got.top_ids) and torch.equal(want.top_logp, got.top_logp)
    assert bool((got.top_logp[:, -1] == -INF).all()) and bool(torch.isfinite(got.top_logp[:, :68]).all())
    plain = m.item_logprobs(z, k=5)
    none = m.item_logprobs(z, k=5, seen=torch.zeros(2, 0, dtype=torch.long, device=dev))
    # the scores' rows are 72 columns apart and the masked copy's 70, so the copy's second row is cut into other
    # chunks and its sum is taken in another order: each is within close_logp's bound of the exact value, and
    # the two of each other within twice that
    assert torch.equal(plain.top_ids, none.top_ids)
    d = (plain.top_logp.double() - none.top_logp.double()).abs()
    assert bool((d <= 2 * (160 * U + 4 * U * plain.top_logp.double().abs())).all())
    with pytest.raises(ValueError):
        m.item_logprobs(z, k=5, seen=torch.zeros(3, 1, dtype=torch.long, device=dev))
    with pytest.raises(ValueError):
        m.distill_loss(torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.long), labels=torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError):
        m.distill_loss(torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.long),
                       candidates=torch.zeros(2, 3, dtype=torch.long))


@pytest.mark.parametrize("M,N", [(2100, 50265), (110000, 1000)])
def test_large_gradients_are_those_of_their_parts(dev, M, N):
    """A gradient larger than the caches hold is written another way: bit by bit that of a few of its rows."""
    x = logits_of(dev, torch.bfloat16, M, N, 7)
    tok = torch.randint(0, N, (M, 2), device=dev)
    g, gh = torch.randn(M, 2, device=dev), torch.randn(M, device=dev)
    r = ops.token_logprobs(x, tok, want_entropy=True, want_stats=True)
    d = ops.token_logprobs_bwd(x, r.stats, tok, g, r.entropy, gh)
    for lo in (0, M - 40):
        p = slice(lo, lo + 40)
        part = ops.token_logprobs_bwd(x[p], r.stats[p], tok[p], g[p], r.entropy[p], gh[p])
        assert torch.equal(d[p], part)
        want, size = ref_grad(x[p], 1.0, tok[p], g[p], gh[p])
        close_grad(part, want, size)


def _every_other(t):
    """t's numbers in every other element of a larger buffer."""
    buf = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=t.device)
    buf[..., ::2] = t
    return buf[..., ::2]


@pytest.mark.parametrize("N", [50, 4100])
def test_saved_tensor_hooks_that_move_the_lists(dev, N):
    """Hooks that hand every saved tensor back with gaps between its elements: the same gradient; hooks that leave them
    on the host: an error."""
    x = logits_of(dev, torch.float32, 5, N, 3)
    ids = torch.randint(0, N, (5, 4), device=dev)
    tl = torch.randn(5, 4, device=dev)
    lists = [lambda y: sum(t.sum() for t in train.token_logprobs_train(y, ids, 1.3)),
             lambda y: train.topk_distill_train(y, tl, ids, 2.0)]
    for fn in lists:
        leaf = x.clone().requires_grad_()
        want, = torch.autograd.grad(fn(leaf), leaf)
        with torch.autograd.graph.saved_tensors_hooks(_every_other, lambda t: t):
            out = fn(leaf)
        got, = torch.autograd.grad(out, leaf)
        assert torch.equal(got, want)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
            out = fn(leaf)
        with pytest.raises(ValueError):
            torch.autograd.grad(out, leaf)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(dev)):
            out = fn(leaf)
        got, = torch.autograd.grad(out, leaf)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [40, 5000, 100000])
def test_gradient_at_inverse_temperatures_next_to_the_largest(dev, dt, N):
    """it = 1e38 and weights that sum to 6: it times their sum is past fp32's range, every gradient is within it: 0
    where p = 0 and nothing is listed, +-2e38 at the listed entries."""
    x = logits_of(dev, dt, 3, N, N)
    x[:, N // 2] = 40.0
    tokens = torch.tensor([[N // 2, N // 2, 1]] * 3, device=dev)
    w, wh = torch.full((3, 3), 2.0, device=dev), torch.ones(3, device=dev)
    leaf = x.clone().requires_grad_()
    logp, h = train.token_logprobs_train(leaf, tokens, inv_temp=1e38)
    both, = torch.autograd.grad((logp, h), leaf, (w, wh), retain_graph=True)
    only, = torch.autograd.grad(logp, leaf, w)
    for d, gh in ((both, wh), (only, torch.zeros_like(wh))):
        want, size = ref_grad(x, 1e38, tokens, w, gh)
        assert float(want.abs().max()) < 2.1e38 and bool((want != 0).sum(1).eq(2).all())
        close_grad(d, want, size)
        assert int((d != 0).sum()) == 6
