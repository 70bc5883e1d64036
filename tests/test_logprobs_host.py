"""Refusals of the log-probability, distillation and 4-bit entry points that need no device: each comes back as
an error with a message before anything is launched, and calls on nothing succeed."""
import ctypes

import pytest
import torch

from recformer_amd import Mxfp4Catalog, _lib, ops, train

A = 1 << 12  # an address that is never read


def err(rc):
    assert rc != 0
    return _lib.load().rf_last_error().decode()


def fwd(dtype=0, M=2, N=50, x=A, ld=50, it=1.0, tok=A, C=1, k=0, logp=A, ent=None, tv=None, ti=None, st=None, ws=None):
    return _lib.load().rf_token_logprobs_fwd(dtype, M, N, x, ld, it, tok, C, -100, k, logp, ent, tv, ti, st, ws, None)


def test_token_logprobs_refusals():
    assert "dtype" in err(fwd(dtype=7))
    assert "shape" in err(fwd(N=0))
    assert "shape" in err(fwd(ld=49))
    for it in (0.0, -1.0, float("nan"), float("inf")):
        assert "temperature" in err(fwd(it=it))
    assert "entries" in err(fwd(C=1025))
    for k in (51, 257, -1):
        assert "k=" in err(fwd(N=300 if k == 257 else 50, ld=300, k=k, tv=A, ti=A))
    assert "null" in err(fwd(x=None))
    assert "null" in err(fwd(tok=None))
    assert "null" in err(fwd(k=3))
    assert "misaligned" in err(fwd(x=A + 2))
    assert "workspace" in err(fwd(M=1, N=1 << 20, ld=1 << 20))
    assert "workspace" in err(fwd(M=1, N=1 << 20, ld=1 << 20, ws=A + 8))
    assert fwd(M=0) == 0


def test_gradient_refusals():
    lib = _lib.load()

    def bwd(x=A, ld=56, st=A, tok=A, g=A, ent=None, ge=None, d=A + 64, ldd=56):
        return lib.rf_token_logprobs_bwd(1, 2, 50, x, ld, 1.0, st, tok, 1, -100, g, ent, ge, d, ldd, None)

    assert "entropy" in err(bwd(ge=A))
    assert "aligned" in err(bwd(d=A + 66))
    assert "aligned" in err(bwd(ldd=51))
    assert "null" in err(bwd(st=None))
    assert "shape" in err(bwd(ldd=48))

    def dist(K=2, t=A, rows=A, st=A, loss=None, coef=None):
        return lib.rf_topk_distill_fwd(0, 2, 50, A, 50, 1.0, t, A, K, 1.0, rows, st, loss, coef, None, None)

    assert "K=0" in err(dist(K=0))
    assert "entries" in err(dist(K=1025))
    assert "null" in err(dist(t=None))
    assert "together" in err(dist(loss=A))
    assert "null" in err(lib.rf_topk_distill_bwd(0, 2, 50, A, 50, 1.0, A, A, A, 2, None, A, A, 50, None))


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.rf_logprobs_workspace(1, 4915, 50265, 20) == 0  # a row a workgroup
    assert lib.rf_logprobs_workspace(0, 0, 50, 5) == 0
    n = lib.rf_logprobs_workspace(0, 1, 1000003, 256)
    assert n > 0 and n % (16 + 8 * 256) == 0
    # a row of 2^31 - 17 columns still has a plan
    assert lib.rf_logprobs_workspace(0, 1, 2 ** 31 - 17, 256) >= (2 ** 31 // 32768) * (16 + 8 * 256)


def test_sizes_past_a_launch_are_refused():
    """Column numbers fit 32 bits with a workgroup's reach past the row's end, a launch has at most 2^32 - 1
    threads, and the plan of very many rows is made in 64 bits."""
    lib = _lib.load()
    top = 2 ** 31 - 1
    assert "shape" in err(fwd(N=top - 2 ** 16 + 1, ld=top))
    assert "too many" in err(fwd(M=top, N=5, ld=5))
    assert "too many" in err(fwd(M=2 ** 22, N=200, ld=200, k=129, tv=A, ti=A))
    assert "too many" in err(lib.rf_token_logprobs_bwd(1, 2 ** 26, 50, A, 50, 1.0, A, A, 1, -100, A, None, None, A, 50,
                                                       None))
    assert lib.rf_logprobs_workspace(0, top, 50, 5) == 0
    assert lib.rf_logprobs_workspace(0, top - 100, 100000, 0) > 0
    assert "too many" in err(lib.rf_mxfp4_quantize(0, 2 ** 26, 512, A, 512, 1e-8, A, A, None, None))
    assert "too many" in err(lib.rf_mxfp4_dequantize(0, 2 ** 28, 512, A, A, A, 512, None))
    assert "too many" in err(lib.rf_mxfp4_gemm(0, top, 1 << 24, 32, A, A, A, A, None, None, None, 1.0, A, 1 << 24,
                                               None))


def test_inverse_temperatures_whose_exponent_overflows_are_refused():
    assert "temperature" in err(fwd(it=2.5e38))  # times log2(e) it is inf, and 0 * inf no number


def test_mxfp4_refusals():
    lib = _lib.load()
    assert "dtype" in err(lib.rf_mxfp4_quantize(3, 1, 32, A, 32, 1e-8, A, A, None, None))
    assert "shape" in err(lib.rf_mxfp4_quantize(0, 1, 0, A, 32, 1e-8, A, A, None, None))
    assert "shape" in err(lib.rf_mxfp4_quantize(0, 1, 32, A, 31, 1e-8, A, A, None, None))
    assert "misaligned" in err(lib.rf_mxfp4_quantize(0, 1, 32, A, 32, 1e-8, A + 4, A, None, None))
    assert "null" in err(lib.rf_mxfp4_quantize(0, 1, 32, None, 32, 1e-8, A, A, None, None))
    assert "shape" in err(lib.rf_mxfp4_dequantize(0, 1, 32, A, A, A, 31, None))

    def gemm(M=2, N=8, K=32, ac=A, ra=None, rw=None, bias=None, C=A, ldc=8, dt=0):
        return lib.rf_mxfp4_gemm(dt, M, N, K, ac, A, A, A, bias, ra, rw, 1.0, C, ldc, None)

    assert "together" in err(gemm(ra=A))
    assert "aligned" in err(gemm(ac=A + 8))
    assert "aligned" in err(gemm(C=A + 4))
    assert "aligned" in err(gemm(ldc=9))
    assert "aligned" in err(gemm(bias=A + 4))
    assert "shape" in err(gemm(ldc=7))
    assert "64 MB" in err(gemm(ldc=1 << 25))
    assert gemm(M=0) == 0 and gemm(N=0) == 0


def test_tensors_on_the_cpu_are_refused():
    x, ids = torch.zeros(2, 64), torch.zeros(2, dtype=torch.long)
    q = ops.Mxfp4(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), 64)
    assert q.rows == 2
    for call in (lambda: ops.token_logprobs(x, ids), lambda: train.token_logprobs_train(x, ids),
                 lambda: train.topk_distill_train(x, x, ids[:, None]), lambda: ops.mxfp4_quantize(x),
                 lambda: ops.mxfp4_dequantize(q), lambda: ops.mxfp4_gemm(x, q), lambda: Mxfp4Catalog.from_items(x),
                 lambda: Mxfp4Catalog(q, torch.ones(2)).scores(x, 1.0)):
        with pytest.raises(_lib.RecformerHipError):
            call()
    with pytest.raises(ValueError):
        Mxfp4Catalog(q, torch.ones(3))


def test_signatures_take_what_the_header_declares():
    """The argument counts of the new entry points, header against binding."""
    import os
    import re
    txt = open(os.path.join(os.path.dirname(__file__), "..", "include", "recformer_hip.h")).read()
    for name in ("rf_token_logprobs_fwd", "rf_token_logprobs_bwd", "rf_topk_distill_fwd", "rf_topk_distill_bwd",
                 "rf_logprobs_workspace", "rf_mxfp4_quantize", "rf_mxfp4_dequantize", "rf_mxfp4_gemm"):
        args = re.search(name + r"\(([^;]*)\);", txt).group(1).split(",")
        types = _lib.SIGNATURES[name][1]
        assert len(args) == len(types), name
        for a, t in zip(args, types):
            ptr = "*" in a or "rf_stream_t" in a
            want = (ctypes.c_void_p if ptr else ctypes.c_float if "float" in a else
                    ctypes.c_int64 if "int64_t" in a else ctypes.c_int)
            assert t is want, (name, a)


class Ctx:
    """An autograd context whose saved tensors may be put in other places, as hooks on saved tensors do."""

    needs_input_grad = (True, False, False, False)

    def save_for_backward(self, *t):
        self.saved_tensors = t

    def set_materialize_grads(self, on):
        pass


class OnDevice(torch.Tensor):
    """A host tensor that says it is on device 0."""

    @staticmethod
    def __new__(cls, t):
        return t.as_subclass(cls)

    def get_device(self):
        return 0


def _saved_by_forward(monkeypatch, kind, put=lambda t: t):
    """The context that a forward on 3 rows of 40 leaves, and the calls that its backward makes; no kernel runs."""
    calls = []
    x = put(torch.randn(3, 40))
    ids = put(torch.arange(12).view(3, 4))
    monkeypatch.setattr(ops, "_dev", lambda *ts: None)
    monkeypatch.setattr(ops, "_logprobs", lambda *a: ops.TokenLogprobs(put(torch.zeros(3, 4)), put(torch.zeros(3)), None,
                                                                       None, put(torch.arange(12.0).view(3, 4))))
    monkeypatch.setattr(ops, "_distill", lambda *a: (put(torch.zeros(())), put(torch.arange(16.0))))
    monkeypatch.setattr(ops, "_logprobs_grad", lambda rows, *a: calls.append((rows, *a)))
    monkeypatch.setattr(ops, "_distill_grad", lambda rows, *a: calls.append((rows, *a)))
    ctx = Ctx()
    if kind == "logprobs":
        train._TokenLogprobs.forward(ctx, x, ids, 1.0, -100)
        back = lambda: train._TokenLogprobs.backward(ctx, torch.ones(3, 4), torch.ones(3))
    else:
        train._TopkDistill.forward(ctx, x, put(torch.randn(3, 4)), ids, 2.0)
        back = lambda: train._TopkDistill.backward(ctx, torch.ones(()))
    return ctx, calls, back


def _strided(t):
    """The same numbers, every other element of a larger buffer."""
    buf = torch.full((*t.shape[:-1], 2 * t.shape[-1]), -1, dtype=t.dtype)
    buf[..., ::2] = t
    return buf[..., ::2]


@pytest.mark.parametrize("kind", ["logprobs", "distill"])
def test_saved_lists_with_other_strides_reach_the_gradient_in_order(monkeypatch, kind):
    ctx, calls, back = _saved_by_forward(monkeypatch, kind)
    with torch.no_grad():
        back()
        saved = ctx.saved_tensors
        ctx.saved_tensors = tuple(_strided(t) for t in saved)  # the logits are no row-major view either
        back()
    (_, *want), (rows, *got) = calls
    assert rows[:3] == (0, 3, 40) and rows[3] == got[0].data_ptr() and rows[4] == 40
    for a, b in zip(want, got):
        if isinstance(a, torch.Tensor):
            assert torch.equal(a, b) and b.is_contiguous()
    assert all(not t.is_contiguous() for t in ctx.saved_tensors)


@pytest.mark.parametrize("kind", ["logprobs", "distill"])
def test_saved_tensors_left_elsewhere_are_refused(monkeypatch, kind):
    """On another device, or of another type or shape: an error, before anything is launched by their address."""
    ctx, calls, back = _saved_by_forward(monkeypatch, kind, OnDevice)
    saved = ctx.saved_tensors
    with torch.no_grad():
        back()
        assert len(calls) == 1
        for i, t in enumerate(saved):
            for bad in (t.as_subclass(torch.Tensor), t.to(torch.float64), t[:-1], t.repeat_interleave(2)):
                ctx.saved_tensors = saved[:i] + (bad,) + saved[i + 1:]
                with pytest.raises(ValueError):
                    back()
        for bad in (saved[0].t(), saved[0].reshape(6, 20), saved[0].reshape(3, 8, 5)):
            ctx.saved_tensors = (bad, *saved[1:])
            with pytest.raises(ValueError):
                back()
    assert len(calls) == 1


def test_mxfp4_sizes_past_the_c_ints_are_refused(monkeypatch):
    """2^32 rows would be 0 rows there, 2^32 + 32 columns a row of 32: refused before anything is allocated."""
    monkeypatch.setattr(ops, "_dev", lambda *ts: None)
    for rows, k in ((2 ** 31, 32), (2 ** 32, 32), (2 ** 32 + 3, 1), (1, 2 ** 24 + 1), (2, 2 ** 32 + 32)):
        x = torch.empty(rows, k, dtype=torch.bfloat16, device="meta")
        kb = -(-k // 32)
        q = ops.Mxfp4(torch.empty(rows, kb * 16, dtype=torch.uint8, device="meta"),
                      torch.empty(rows, kb, dtype=torch.uint8, device="meta"), k)
        one = ops.Mxfp4(torch.empty(1, kb * 16, dtype=torch.uint8), torch.empty(1, kb, dtype=torch.uint8), k)
        for call in (lambda: ops.mxfp4_quantize(x), lambda: ops.mxfp4_quantize(x, want_rnorm=True),
                     lambda: ops.mxfp4_dequantize(q), lambda: ops.mxfp4_gemm(x, one), lambda: ops.mxfp4_gemm(q, one),
                     lambda: Mxfp4Catalog.from_items(x)):
            with pytest.raises(ValueError, match="2\\^31 rows"):
                call()


def test_product_tiles_are_counted_in_64_bits():
    """Rows next to 2^31: the count of row tiles stays positive, so that too many tiles are seen as such."""
    lib = _lib.load()
    for M in (2 ** 31 - 127, 2 ** 31 - 1):
        assert "too many tiles" in err(lib.rf_mxfp4_gemm(0, M, 1 << 24, 32, A, A, A, A, None, None, None, 1.0, A, 1 << 24,
                                                         None))


def test_weights_without_their_tokens_are_refused(monkeypatch):
    """Without tokens the log probabilities' weights would be left out of the gradient."""
    monkeypatch.setattr(ops, "_dev", lambda *ts: None)
    monkeypatch.setattr(ops, "_logprobs_grad", lambda *a: a)
    x, stats, g = torch.zeros(2, 8), torch.zeros(2, 4), torch.ones(2)
    with pytest.raises(ValueError, match="tokens"):
        ops.token_logprobs_bwd(x, stats, None, g)
    with pytest.raises(ValueError, match="tokens"):
        ops.token_logprobs_bwd(x, stats, None, g, g, g)
    ops.token_logprobs_bwd(x, stats, None, None, g, g)


def test_temperatures_whose_square_leaves_fp32_are_refused(monkeypatch):
    """temp^2 is 0 or inf there: a loss and gradient of 0, or NaN."""
    monkeypatch.setattr(train._TopkDistill, "apply", lambda *a: a[-1])
    x, ids = torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.long)
    for bad in (1e-30, 9e-19, 1.1e18, 1e20, 0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            train.topk_distill_train(x, x[:, :1], ids, bad)
    for temp in (1e-18, 1, 2.5, 1e18):
        assert train.topk_distill_train(x, x[:, :1], ids, temp) == temp
        assert 0 < ctypes.c_float(temp * temp).value < float("inf")


class Scorer:
    """The scores of 2 users and 6 items in the place of a model's."""

    def similarity_score(self, z):
        return torch.arange(12, dtype=torch.float32).view(2, 6)


@pytest.fixture
def masked_scores(monkeypatch):
    from recformer_amd.models import RecformerForSeqRec
    monkeypatch.setattr(ops, "token_logprobs", lambda scores, *a, **kw: scores)
    return lambda seen: RecformerForSeqRec.item_logprobs(Scorer(), None, seen=seen)


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_history_under_another_default_type(masked_scores, dtype):
    was = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        got = masked_scores(torch.tensor([[5, -1], [0, 0]]))
    finally:
        torch.set_default_dtype(was)
    want = Scorer().similarity_score(None)
    want[0, 5] = want[1, 0] = -float("inf")
    assert got.dtype == torch.float32 and torch.equal(got, want)


def test_history_that_is_no_list_of_ids_is_refused(masked_scores):
    """A mask over the items would be taken for the ids 0 and 1, and fractions would be cut."""
    for seen in (torch.ones(2, 6, dtype=torch.bool), torch.ones(2, 1), torch.ones(2, 1, dtype=torch.bfloat16)):
        with pytest.raises(TypeError):
            masked_scores(seen)
    for dtype in (torch.uint8, torch.int16, torch.int32, torch.int64):
        assert bool(torch.isneginf(masked_scores(torch.tensor([[5], [0]], dtype=dtype))[[0, 1], [5, 0]]).all())


@pytest.mark.parametrize("dtype,n", [(torch.uint8, 10000), (torch.int8, 200), (torch.int16, 50265)])
def test_history_ids_of_a_type_narrower_than_the_catalog(masked_scores, monkeypatch, dtype, n):
    monkeypatch.setattr(Scorer, "similarity_score", lambda self, z: torch.zeros(2, n))
    got = masked_scores(torch.tensor([[100, 3], [0, 127]], dtype=dtype))
    assert torch.isneginf(got).nonzero().tolist() == [[0, 3], [0, 100], [1, 0], [1, 127]]
