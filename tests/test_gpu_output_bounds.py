"""What the log-probability, distillation and 4-bit kernels write: every output lies in a larger buffer of one
number, and all of that buffer outside of the output is still that number afterwards. The outputs themselves
equal, bit by bit, those that the Python calls allocate."""
import pytest
import torch

from recformer_amd import _lib, ops
from recformer_amd._lib import check
from recformer_amd.ops import RF_BF16, dtype_code

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
MARK = 77


class Guarded:
    """A (rows, cols) output within a buffer of MARKs: `lead` elements and a row before it, rows of stride `ld`, and a
    row behind it."""

    def __init__(self, dev, dtype, rows, cols, ld=None, lead=0):
        ld = cols if ld is None else ld
        at = -(-max(ld, 1) // 64) * 64  # 16-byte aligned, but for lead
        self.buf = torch.full((at + lead + (rows + 1) * ld + 64,), MARK, dtype=dtype, device=dev)
        self.view = self.buf.as_strided((rows, cols), (ld, 1), at + lead)
        self.ptr = self.view.data_ptr()

    def get(self):
        """The output, after a look at everything around it."""
        out = self.view.clone()
        self.view.fill_(MARK)
        assert bool((self.buf == MARK).all())
        return out


def stream():
    return torch.cuda.current_stream().cuda_stream


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), 12345.0), torch.nan_to_num(b.double(), 12345.0))


def logits_of(dev, dt, M, N, lead, pad):
    """Logits and a gradient's place of the same layout."""
    V = 16 // (torch.finfo(dt).bits // 8)
    ld = N + pad
    x = Guarded(dev, dt, M, N, ld, lead)
    x.view.copy_((torch.randn(M, N, device=dev) * 3).to(dt))
    d = Guarded(dev, dt, M, N, ld + V, lead)
    return x.view, ld, d, ld + V


# one wave, 256 threads, several slices; rows that start off the 16-byte border and end anywhere
SIZES = [(5, 1), (5, 50), (3, 1999), (3, 4103), (2, 20001), (2, 140003)]


@pytest.mark.parametrize("lead,pad", [(0, 0), (1, 3), (3, 8), (7, 5)])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N", SIZES)
def test_log_probabilities_and_their_gradient(dev, dt, M, N, lead, pad):
    lib, code = _lib.load(), dtype_code(dt)
    x, ld, d, ldd = logits_of(dev, dt, M, N, lead, pad)
    tokens = torch.randint(0, N, (M, 3), device=dev)
    tokens[:, 2] = N - 1
    tokens[0, 1] = -100
    k = min(N, 20)
    f32 = torch.float32
    logp, ent = Guarded(dev, f32, M, 3), Guarded(dev, f32, M, 1)
    tv, ti = Guarded(dev, f32, M, k), Guarded(dev, torch.int64, M, k)
    stats = Guarded(dev, f32, M, 4)
    ws = Guarded(dev, torch.uint8, 1, lib.rf_logprobs_workspace(code, M, N, k))
    check(lib.rf_token_logprobs_fwd(code, M, N, x.data_ptr(), ld, 0.7, tokens.data_ptr(), 3, -100, k, logp.ptr, ent.ptr,
                                    tv.ptr, ti.ptr, stats.ptr, ws.ptr, stream()), "rf_token_logprobs_fwd")
    ws.get()
    want = ops.token_logprobs(x, tokens, k=k, inv_temp=0.7, want_entropy=True, want_stats=True)
    st, en = stats.get(), ent.get()
    assert same(logp.get(), want.logp) and same(en[:, 0], want.entropy) and same(tv.get(), want.top_logp)
    assert torch.equal(ti.get(), want.top_ids) and same(st, want.stats)
    g, gh = torch.randn(M, 3, device=dev), torch.randn(M, device=dev)
    for weight in (None, gh):
        check(lib.rf_token_logprobs_bwd(code, M, N, x.data_ptr(), ld, 0.7, st.data_ptr(), tokens.data_ptr(), 3, -100,
                                        g.data_ptr(), en.data_ptr(), None if weight is None else gh.data_ptr(), d.ptr,
                                        ldd, stream()), "rf_token_logprobs_bwd")
        ref = ops.token_logprobs_bwd(x, st, tokens, g, None if weight is None else want.entropy, weight, 0.7)
        assert same(d.get(), ref)


@pytest.mark.parametrize("K", [2, 100])
@pytest.mark.parametrize("lead,pad", [(0, 0), (3, 5), (5, 8)])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N", SIZES)
def test_distillation_and_its_gradient(dev, dt, M, N, lead, pad, K):
    lib, code = _lib.load(), dtype_code(dt)
    x, ld, d, ldd = logits_of(dev, dt, M, N, lead, pad)
    ids, tl = torch.randint(0, N, (M, K), device=dev), torch.randn(M, K, device=dev)
    ids[:, 0] = N - 1
    ids[0, 1] = -1
    f32 = torch.float32
    rows, stats = Guarded(dev, f32, M, 1), Guarded(dev, f32, M, 4)
    loss, coef = Guarded(dev, f32, 1, 1), Guarded(dev, f32, 1, 1)
    ws = Guarded(dev, torch.uint8, 1, lib.rf_logprobs_workspace(code, M, N, 0))
    check(lib.rf_topk_distill_fwd(code, M, N, x.data_ptr(), ld, 0.5, tl.data_ptr(), ids.data_ptr(), K, 4.0, rows.ptr,
                                  stats.ptr, loss.ptr, coef.ptr, ws.ptr, stream()), "rf_topk_distill_fwd")
    ws.get()
    r, s, mean, c = ops.topk_distill(x, tl, ids, 0.5, 4.0)
    st, co = stats.get(), coef.get()
    assert same(rows.get()[:, 0], r) and same(st, s) and same(loss.get()[0, 0], mean) and same(co[0, 0], c)
    g = torch.full((1,), 3.0, device=dev)
    check(lib.rf_topk_distill_bwd(code, M, N, x.data_ptr(), ld, 0.5, st.data_ptr(), tl.data_ptr(), ids.data_ptr(), K,
                                  g.data_ptr(), co.data_ptr(), d.ptr, ldd, stream()), "rf_topk_distill_bwd")
    assert same(d.get(), ops.topk_distill_bwd(x, s, tl, ids, g, c, 0.5))


def test_gradient_larger_than_the_caches(dev):
    """Written past them: 2200 rows of 50265 16-bit columns, 5 elements off the border."""
    lib, M, N = _lib.load(), 2200, 50265
    x, ld, d, ldd = logits_of(dev, torch.bfloat16, M, N, 5, 2)
    tokens = torch.randint(0, N, (M, 1), device=dev)
    st = ops.token_logprobs(x, tokens, want_stats=True).stats
    g = torch.randn(M, 1, device=dev)
    check(lib.rf_token_logprobs_bwd(RF_BF16, M, N, x.data_ptr(), ld, 1.0, st.data_ptr(), tokens.data_ptr(), 1, -100,
                                    g.data_ptr(), None, None, d.ptr, ldd, stream()), "rf_token_logprobs_bwd")
    got = d.get()
    assert torch.equal(got, ops.token_logprobs_bwd(x, st, tokens, g))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 33), (70, 100), (9, 770), (5, 4095)])
def test_quantise_and_back(dev, dt, M, K):
    lib, code, kb = _lib.load(), dtype_code(dt), (K + 31) // 32
    x = Guarded(dev, dt, M, K, K + 3, 1).view
    x.copy_(torch.randn(M, K, device=dev).to(dt))
    codes, scales = Guarded(dev, torch.uint8, M, kb * 16), Guarded(dev, torch.uint8, M, kb)
    rn = Guarded(dev, torch.float32, M, 1)
    check(lib.rf_mxfp4_quantize(code, M, K, x.data_ptr(), K + 3, 1e-8, codes.ptr, scales.ptr, rn.ptr, stream()),
          "rf_mxfp4_quantize")
    q, norm = ops.mxfp4_quantize(x, want_rnorm=True)
    assert torch.equal(codes.get(), q.codes) and torch.equal(scales.get(), q.scales) and same(rn.get()[:, 0], norm)
    for lead, pad in ((0, 0), (0, 8), (1, 3), (4, 7)):
        out = Guarded(dev, dt, M, K, K + pad, lead)
        check(lib.rf_mxfp4_dequantize(code, M, K, q.codes.data_ptr(), q.scales.data_ptr(), out.ptr, K + pad, stream()),
              "rf_mxfp4_dequantize")
        assert same(out.get(), ops.mxfp4_dequantize(q, dt))


# every kernel and its edges: up to 64 rows with one and four tiles a wave, tiles of 128 x 128, several a workgroup
PRODUCTS = [(1, 1, 32), (3, 70, 96), (17, 129, 64), (33, 500, 160), (64, 32801, 64), (5, 33003, 96), (65, 127, 64),
            (129, 257, 96), (200, 300, 768), (130, 131, 1000), (4200, 4101, 128)]


@pytest.mark.parametrize("lead,pad", [(0, 0), (4, 4), (8, 12)])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(dev, dt, M, N, K, lead, pad):
    lib = _lib.load()
    a, w = ops.mxfp4_quantize(torch.randn(M, K, device=dev)), ops.mxfp4_quantize(torch.randn(N, K, device=dev))
    bias = torch.randn(N, device=dev)
    ldc = (N + 3) // 4 * 4 + pad
    c = Guarded(dev, dt, M, N, ldc, lead)
    check(lib.rf_mxfp4_gemm(dtype_code(dt), M, N, K, a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(),
                            w.scales.data_ptr(), bias.data_ptr(), None, None, 1.0, c.ptr, ldc, stream()),
          "rf_mxfp4_gemm")
    assert same(c.get(), ops.mxfp4_gemm(a, w, bias, dt))
