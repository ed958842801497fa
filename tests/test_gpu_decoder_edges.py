"""Decoder-block operators at the edges of their contracts: non-finite operands, rows that see nothing, calls that tests of
ordinary shapes do not make (B200 only)."""
import math

import pytest

import decoder_ref as ref
from test_gpu_decoder import Attention, workspace

pytestmark = pytest.mark.gpu


# ---- attention: non-finite keys and values -------------------------------------------------------------------------
FORMS = {"prompt": dict(q=130, dim=64), "tokens": dict(q=5, dim=64), "rows": dict(q=5, dim=64, pad=1), "rows, long": dict(q=130, dim=64, pad=1)}


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("form", FORMS)
def test_attention_rows_without_a_key_are_zero_whatever_the_values_hold(cuda, form, value):
    """Three keys behind more queries than that: the first queries see none, and give zeros and lse -infinity although the
    keys they do not see have values that are not finite."""
    f = dict(FORMS[form])
    q = f.pop("q")
    a = Attention(cuda, [q], [3], 8, 2, type="f16", causal=True, slab=16, **f)
    a.v[0] = value
    for w in (workspace(cuda), None):
        a.out.fill_(7)
        a.call(w)
        cuda.cuda.synchronize()
        got = a.out[:, :8 * a.dim]
        assert bool((got[:q - 3] == 0).all()) and bool((a.lse[:q - 3] == -math.inf).all())
        assert not bool(got[q - 3:].isfinite().any())
        want_lse, tol_lse = ref.attention(a.q, a.k, a.v, a.q_start, a.k_start, a.k_len, a.scale, True, "f16")[1::2]
        assert bool(((a.lse - want_lse).abs()[q - 3:] <= tol_lse[q - 3:]).all())


@pytest.mark.parametrize("form", FORMS)
def test_attention_keys_that_score_minus_infinity(cuda, form):
    """Every key of the sequence scores -infinity: no weight is left, zeros and lse -infinity, also with infinite values."""
    f = dict(FORMS[form])
    q = f.pop("q")
    a = Attention(cuda, [q], [200], 8, 2, type="bf16", causal=False, **f)
    a.q.abs_().add_(0.5)
    a.k.fill_(-math.inf)
    a.v[7] = math.inf
    a.call(workspace(cuda))
    cuda.cuda.synchronize()
    assert bool((a.out[:, :8 * a.dim] == 0).all()) and bool((a.lse == -math.inf).all())


@pytest.mark.parametrize("q,heads,kv_heads", [(65, 8, 8), (193, 8, 8), (22, 24, 8)])
def test_attention_rows_that_are_not_stored_cost_nothing(cuda, q, heads, kv_heads):
    """A tile's rows behind the last sequence hold zeros or NaN: the same results bit for bit, and no more time.  Without the
    rule that only stored rows ask for a rescale the call with NaN takes 1.13 times as long; the least of many calls in turn
    repeats itself to one part in a hundred."""
    a = Attention(cuda, [q], [16384], heads, kv_heads, 128, "f16", False, behind=128)
    stream = cuda.cuda.current_stream().cuda_stream
    best, out = {}, {}
    for _ in range(40):
        for fill in (0.0, math.nan):
            a.q[q:] = fill
            begin, end = cuda.cuda.Event(enable_timing=True), cuda.cuda.Event(enable_timing=True)
            begin.record()
            a.call(stream=stream)
            end.record()
            end.synchronize()
            key = "zero" if fill == 0 else "nan"
            best[key] = min(best.get(key, math.inf), begin.elapsed_time(end))
            out[key] = a.out[:q].clone()
    assert cuda.equal(out["zero"], out["nan"])
    a.check()
    assert best["nan"] <= 1.05 * best["zero"], best


# ---- 8-bit products ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,N,K", [(1, 4096, 16), (16, 512, 1024), (64, 300, 400), (130, 1234, 1040), (65, 64, 128)])
def test_i8gemm_launches_one_behind_the_other(cuda, M, N, K):
    """CTAs that follow each other on an SM: hundreds of launches with nothing between them give what the first one gives,
    with fewer blocks of k than stages and with more."""
    from tacker_b200 import ops

    g = cuda.Generator(device="cuda")
    g.manual_seed(M)
    a, b = (cuda.randint(-128, 128, (r, K), generator=g, device="cuda", dtype=cuda.int8) for r in (M, N))
    sa, sb = cuda.rand(M, generator=g, device="cuda"), cuda.rand(N, generator=g, device="cuda")
    outs = [cuda.full((M, N), 7.0, device="cuda") for _ in range(300)]
    cuda.cuda.synchronize()
    for o in outs:
        ops.i8gemm(a.data_ptr(), K, sa.data_ptr(), b.data_ptr(), K, sb.data_ptr(), 0, o.data_ptr(), N, 0, M, N, K)
    cuda.cuda.synchronize()
    want, tol = ref.i8gemm(a, sa, b, sb, None, "f32")
    assert bool(((outs[0].double() - want).abs() <= tol).all())
    assert all(cuda.equal(o, outs[0]) for o in outs)
    assert ops.device_status() == 0


# ---- bounded waits -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("q", [65, 200])
def test_attention_waits_that_span_an_item_outlast_their_budget(cuda, q):
    """Items of 2048 key tiles take about 3 ms; with a budget of 1 ms no wait may run out as long as its tiles go on.  One
    row tile (the other's warps wait through the whole item) and two."""
    from tacker_b200 import ops

    keys = 1 << 18
    a = Attention(cuda, [q], [keys], 1, 1, 128, "bf16", False, poison=False)
    assert ops.device_status() == 0
    ops.set_option("wait_budget_us", 1000)
    try:
        a.call()
        cuda.cuda.synchronize()
        assert ops.device_status() == 0
    finally:
        ops.set_option("wait_budget_us", 1000000)
    a.check()


# ---- the residual stream in place ----------------------------------------------------------------------------------
@pytest.mark.parametrize("cols", [4096, 768, 59])
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("y_over,h_over", [("a", None), ("x", None), (None, "a"), (None, "x"), ("a", "x"), ("x", "a")])
def test_norm_in_place(cuda, cols, type, y_over, h_over):
    """y and h over a or x: what separate buffers get, bit for bit."""
    from tacker_b200 import ops

    rows, t, code = 700, ref.TYPES[type], ref.CODES[type]
    g = cuda.Generator(device="cuda")
    g.manual_seed(cols)
    a, x = (cuda.randn(rows, cols, generator=g, device="cuda").to(t) for _ in "ax")
    gamma = cuda.randn(cols, generator=g, device="cuda")

    def call(a, x, y, h):
        ops.norm_residual_rows(a.data_ptr(), code, cols, 1, gamma.data_ptr(), 0, 0, 0, 1, 0.5, x.data_ptr(), cols, y.data_ptr(), cols,
                               code, gamma.data_ptr(), 0, h.data_ptr(), cols, code, 1, 1e-5, rows, cols)
        cuda.cuda.synchronize()

    y, h = cuda.zeros_like(a), cuda.zeros_like(a)
    call(a, x, y, h)
    here = {"a": a.clone(), "x": x.clone(), None: cuda.zeros_like(a)}
    yy, hh = here[y_over], here[h_over]
    call(here["a"], here["x"], yy, hh)
    assert cuda.equal(yy, y) and cuda.equal(hh, h)
