"""Decoder-block operators at the edges of their contracts: non-finite operands, rows that see nothing, calls that tests of
ordinary shapes do not make (B200 only)."""
import math

import pytest

import decoder_ref as ref
from test_gpu_decoder import Attention, Block, at, normal, within, workspace

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


def test_attention_search_for_items_outlasts_the_budget(cuda):
    """Two sequences with tokens among 600000 without: the search for their items, and the blocks that have none, take several
    times the budget of a wait, and no wait runs out."""
    from tacker_b200 import ops

    n, kv_heads, dim = 600_000, 8, 64
    a = Attention(cuda, [200, 130], [200, 130], 8, kv_heads, dim, "f16", True)
    many = [cuda.zeros(n + 1, dtype=cuda.int32, device="cuda") for _ in range(3)]
    many[0][1000:] = 200
    many[0][n:] = 330  # sequence 999 has 200 tokens, the last one 130
    many[1][n - 1] = 200
    many[2][999], many[2][n - 1] = 200, 130
    assert ops.device_status() == 0
    ops.set_option("wait_budget_us", 1000)
    try:
        ops.attention_packed(at(a.q), 8 * dim, at(a.k), 8 * dim, at(a.v), 8 * dim, at(a.out), 8 * dim, at(a.lse), 1, *(at(x) for x in many), n,
                             a.total, a.rows, 200, 200, 8, 8, dim, a.scale, 1)
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


# ---- attention: precision of the forms -----------------------------------------------------------------------------
def two_term_bound(a):
    """(out, bound, out with weights rounded once) of calls with one token per sequence, in binary64.

    Weights enter as p = hi + lo in the values' type: hi is off by half a step of p, lo by half a step of what hi left (or half
    the smallest step there is), so that p is off by half_step^2.  What else is off is fp32: the scores (dim products, the scale,
    the difference to the maximum, the power's 2 ulp) and the sums over n keys, once for the weights and once for the values."""
    torch, U, f = a.torch, ref.U, torch_finfo(a)
    outs, bounds, once = [], [], []
    for i, n in enumerate(a.k_len):
        q = a.q[i].double()
        k, v = (z[a.k_start[i]:a.k_start[i] + n].double().repeat_interleave(a.heads // a.kv_heads, 1) for z in (a.k, a.v))
        s = torch.einsum("hd,jhd->hj", q, k) * a.scale
        size = (torch.einsum("hd,jhd->hj", q.abs(), k.abs()) * a.scale).amax(1)
        m = s.amax(1, keepdim=True)
        e = torch.exp(s - m)
        total = e.sum(1, keepdim=True)
        mix = lambda w, v: torch.einsum("hj,jhd->hd", w / total, v)  # noqa: E731, B023
        out, spread = mix(e, v), mix(e, v.abs())
        off = (a.dim + 4) * U * size + 4 * U * 1.45 * m[:, 0].abs() + 4 * U + n * U
        outs.append(out)
        bounds.append((ref.half_step(a.type) ** 2 + 2 * off[:, None]) * spread + ref.rounding(out, a.type) + n * f.tiny * f.eps / 2 * v.abs().amax())
        once.append(mix(e.to(a.v.dtype).double(), v))
    return (torch.stack(x) for x in (outs, bounds, once))


def torch_finfo(a):
    return a.torch.finfo(ref.TYPES[a.type])


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("dim,pad", [(64, 0), (128, 0), (64, 1)])
@pytest.mark.parametrize("split", [True, False])
def test_attention_tokens_do_not_round_their_weights(cuda, type, dim, pad, split):
    """Values that nearly cancel show what rounding the weights once would cost: more than the bound.  (fp16 with heads of 128
    is only checked against the bound: its fp32 part, (dim + 4) steps of the scores' size, is there larger than half a step of
    fp16, which no test of the result can tell apart.)"""
    k_len = [2, 3, 17, 40, 1024, 700]
    a = Attention(cuda, [1] * len(k_len), k_len, 8, 2, dim, type, True, slab=1024, pad=pad, poison=False)
    first = a.k[:1].clone()
    a.k.mul_(0.05).add_(first)  # scores that are nearly equal
    a.v.copy_(a.v.abs().add(1.0).mul(8))
    a.v[1::2] = -a.v[0::2]
    a.call(workspace(cuda) if split else None)
    cuda.cuda.synchronize()
    want, bound, once = two_term_bound(a)
    got = a.out[:, :a.heads * dim].unflatten(1, (a.heads, dim))
    within(cuda, got, want, bound, "out")
    if type == "bf16" or dim == 64:
        noticed = int(((once - want).abs() > bound).sum())
        assert noticed > 0, "the bound would not notice weights that are rounded once"


@pytest.mark.parametrize("form", ["prompt", "tokens", "tokens, split", "rows"])
@pytest.mark.parametrize("score", [-12.0, -17.5, -20.0])
def test_attention_many_keys_of_little_weight(cuda, form, score):
    """One key that takes almost all of the weight and 60000 that share the rest: weights of e^-12 to e^-20, the last two below
    the steps of fp16, whose values decide the result.

    Bound: as for scores and sums in fp32 everywhere; weights in fp16 half a step each, and at the end of its range half of its
    smallest step, where the largest weight is 2^7 (prompts) or more."""
    n, dim, q = 60001, 64, {"prompt": 70}.get(form, 1)
    a = Attention(cuda, [q], [n], 1, 1, dim, "f16", False, pad=int(form == "rows"), scale=1.0, poison=False)
    a.q.zero_()[:, :, 0] = 1.0
    a.k.zero_()[1:, :, 0] = score
    a.v[0] = 0
    a.v[1:] = a.v[1:] * 100 + 1000
    a.call(workspace(cuda) if form == "tokens, split" else None)
    cuda.cuda.synchronize()
    U, w = ref.U, math.exp(score)
    total = 1 + (n - 1) * w
    v = a.v[:, 0].double()
    want = v[1:].sum(0) * w / total
    spread = v[1:].abs().sum(0) * w / total
    off = ((dim + 4) + 4 * 1.45) * U * abs(score) + 4 * U + n * U
    bound = (ref.half_step("f16") + 2 * off) * spread + ref.rounding(want, "f16") + n * 2.0 ** -25 * 2.0 ** -7 * v.abs().max()
    got = a.out[:, :dim].double()
    within(cuda, got, want.expand_as(got), bound.expand_as(got), "out")
    lse = cuda.full_like(a.lse.double(), math.log(total))
    within(cuda, a.lse, lse, off + 4 * U * lse.abs(), "lse")


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("type,q0,k0", [("bf16", 1.0, 2.0 ** 17), ("bf16", 1.0, 3e7), ("bf16", -1.0, 1e9), ("bf16", 3.0, 1e20), ("bf16", 1.0, 3e37),
                                        ("f16", 1.0, 60000.0), ("f16", 55.0, 60000.0), ("f16", -60000.0, 60000.0)])
def test_attention_scores_of_any_size(cuda, form, type, q0, k0):
    """Two keys whose scores are larger than all others by far, in two different key tiles: each weighs one half, whatever
    their size; and the same with all scores negative."""
    f = dict(FORMS[form])
    q, dim, pad = f["q"], f["dim"], f.get("pad", 0)
    a = Attention(cuda, [q], [200], 8, 2, dim, type, False, pad=pad, scale=1.0)
    for lowest in (False, True):
        a.q.zero_()[:, :, 0] = q0
        a.k.zero_()
        if lowest:  # the others lie further from zero
            a.k[:, :, 0] = -math.copysign(k0, q0)
            a.k[7, :, 0] = a.k[150, :, 0] = -math.copysign(k0 / 2, q0)
        else:
            a.k[7, :, 0] = a.k[150, :, 0] = math.copysign(k0, q0)
        a.call(workspace(cuda))
        cuda.cuda.synchronize()
        score = a.q[0, 0, 0].double() * a.k[7, 0, 0].double()
        v = a.v.double().repeat_interleave(4, 1)
        want = ((v[7] + v[150]) / 2).expand(q, 8, dim)
        # weights are powers 2^(scale s + off) with off rounded to 32 bits: equal for equal scores, but no powers of two, and
        # prompts round them once to the type (half a step each, on both values; the sum is taken before)
        spread = (v[7].abs() + v[150].abs()) / 2
        bound = (8 * ref.U + ref.half_step(type) * (form == "prompt")) * spread + ref.rounding(want, type)
        got = a.out[:, :8 * dim].unflatten(1, (8, dim))
        within(cuda, got, want, bound, "out")
        lse = (score + math.log(2)).expand(q, 8)
        within(cuda, a.lse, lse, 8 * ref.U * lse.abs(), "lse")


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_large_scores_in_some_rows(cuda, type, dim):
    """Rows with scores of ordinary size, of hundreds of thousands and in between side by side in every warp, over several
    key tiles, causal: each by its own rule.

    Scores of size B are exact to B * 2^-24 times the additions, so that a row's weights are off by that: with one element per
    head that is not zero, the score is one product and its scale, exact but for one rounding each."""
    q = 300
    a = Attention(cuda, [q], [700], 4, 2, dim, type, True, scale=1.0)
    size = 4.0 ** (cuda.arange(q, device="cuda") % 10)  # 1 .. 262144
    a.q.zero_()[:, :, 0] = cuda.where(size > 60000, 1.0, size).to(a.q.dtype)[:, None]
    a.q[:, :, 1] = cuda.where(size > 60000, 32768.0, 0.0).to(a.q.dtype)[:, None]
    k = cuda.randn(700, 2, generator=cuda.Generator(device="cuda").manual_seed(3), device="cuda")
    a.k.zero_()[:, :, 0] = k.to(a.k.dtype)
    a.k[:, :, 1] = (k * 8).round().to(a.k.dtype)
    a.call(workspace(cuda))
    cuda.cuda.synchronize()
    want, want_lse, _, _ = ref.attention(a.q, a.k, a.v, a.q_start, a.k_start, a.k_len, 1.0, True, type)
    s = cuda.einsum("thd,jhd->htj", a.q.double(), a.k.double().repeat_interleave(2, 1))
    see = cuda.arange(700, device="cuda")[None] <= cuda.arange(q, device="cuda")[:, None] + 400
    big = s.masked_fill(~see, 0).abs().amax(2).t()
    p = cuda.softmax(s.masked_fill(~see, -math.inf), 2)
    spread = cuda.einsum("htj,jhd->thd", p, a.v.double().abs().repeat_interleave(2, 1))
    # score: two products' sum (2 U), times log2 e and the rounded maximum (2 U), the difference and the power (4 U); n sums
    off = (4 * 1.45 * big + 4 + 700) * ref.U
    bound = (ref.half_step(type) + 2 * off[..., None]) * spread + ref.rounding(want, type) + 700 * 2.0 ** -25 * (type == "f16") * 4.5 * 2.0 ** -7
    got = a.out[:, :4 * dim].unflatten(1, (4, dim))
    within(cuda, got, want, bound, "out")
    within(cuda, a.lse, want_lse, off + 4 * ref.U * want_lse.abs(), "lse")


def test_calls_repeat_themselves_bit_for_bit(cuda):
    """The same inputs again, after other kernels have used the shared memory: the same bits, in every form."""
    ws = workspace(cuda)
    calls = [Attention(cuda, [300, 1, 64], [300, 700, 900], 6, 2, 128, "bf16", True, slab=1000),
             Attention(cuda, [1] * 5, [3, 700, 65, 900, 1], 8, 2, 64, "f16", True, slab=1000),
             Attention(cuda, [70, 3], [70, 90], 4, 2, 40, "f16", True, pad=1, slab=100)]
    for a in calls:
        first = None
        for i in range(6):
            a.out.fill_(7)
            a.call(ws)
            got = a.out.clone(), a.lse.clone()
            first = first or got
            assert cuda.equal(got[0], first[0]) and cuda.equal(got[1], first[1])
            x = cuda.full((512 * (i + 1), 512), math.nan if i % 2 else 100.0, dtype=cuda.float16, device="cuda")
            x @ x[:512]
            Attention(cuda, [130], [130], 7, 7, 128, "f16", False, seed=i).call(ws)


@pytest.mark.parametrize("form", FORMS)
def test_attention_scores_beyond_fp32(cuda, form):
    """One key that scores +infinity for every other query (no number is left for it) and -infinity for the rest (which do
    not notice it)."""
    f = dict(FORMS[form])
    q, dim, pad = f["q"], f["dim"], f.get("pad", 0)
    a = Attention(cuda, [q], [200], 8, 2, dim, "bf16", False, pad=pad)
    a.q.abs_().add_(0.1)
    a.q[1::2] = -a.q[1::2]
    a.k[150] = 3e38
    for w in (workspace(cuda), None):
        a.out.fill_(7)
        a.call(w)
        cuda.cuda.synchronize()
        got = a.out[:, :8 * dim].unflatten(1, (8, dim))
        assert bool(got[0::2].isnan().all()) and not bool(a.lse[0::2].isfinite().any())
        rest = [i for i in range(200) if i != 150]
        want, want_lse, tol, tol_lse = ref.attention(a.q, a.k[rest], a.v[rest], [0, q], [0], [199], a.scale, False, "bf16")
        within(cuda, got[1::2], want[1::2], tol[1::2], "out")
        within(cuda, a.lse[1::2], want_lse[1::2], tol_lse[1::2], "lse")


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("form", FORMS)
def test_attention_values_that_are_not_finite(cuda, form, value):
    """A value that is not finite leaves no finite number in its element of the queries that see it, and touches nothing else:
    not the other elements, not lse, not the other sequences."""
    f = dict(FORMS[form])
    q, dim, pad = f["q"], f["dim"], f.get("pad", 0)
    a = Attention(cuda, [q, q], [200, 150], 8, 2, dim, "f16", False, pad=pad)
    a.v[120, 1, 5] = value
    a.call(workspace(cuda))
    cuda.cuda.synchronize()
    got = a.out[:, :8 * dim].unflatten(1, (8, dim)).clone()
    assert not bool(got[:q, 4:, 5].isfinite().any())
    a.v[120, 1, 5] = 0.0
    want, want_lse, tol, tol_lse = ref.attention(a.q, a.k, a.v, a.q_start, a.k_start, a.k_len, a.scale, False, "f16")
    got[:q, 4:, 5] = want[:q, 4:, 5].to(got.dtype)
    within(cuda, got, want, tol, "out")
    within(cuda, a.lse, want_lse, tol_lse, "lse")


# ---- every combination of types ------------------------------------------------------------------------------------
@pytest.mark.parametrize("a_type", ref.TYPES)
@pytest.mark.parametrize("x_type", ref.TYPES)
@pytest.mark.parametrize("h_type", ref.TYPES)
@pytest.mark.parametrize("rows,cols", [(300, 4096), (37, 264)])
def test_norm_types(cuda, a_type, x_type, h_type, rows, cols):
    from tacker_b200 import ops

    a, x = normal(cuda, 1, rows, cols, type=a_type, scale=3), normal(cuda, 2, rows, cols, type=x_type, scale=2)
    g = [1 + normal(cuda, 3 + i, cols, scale=0.2) for i in range(4)]
    y, h = (cuda.zeros(rows, cols, dtype=ref.TYPES[t], device="cuda") for t in (x_type, h_type))
    ops.norm_residual_rows(at(a), ref.CODES[a_type], cols, 1, at(g[0]), at(g[1]), 0, 0, 1, 0.7, at(x), cols, at(y), cols, ref.CODES[x_type],
                           at(g[2]), at(g[3]), at(h), cols, ref.CODES[h_type], 1, 1e-5, rows, cols)
    cuda.cuda.synchronize()
    wy, wh, ty, th = ref.norm(a, x, None, 1, 0.7, 1, *g, 1, 1e-5, x_type, h_type)
    within(cuda, y, wy, ty, "y")
    within(cuda, h, wh, th, "h")


@pytest.mark.parametrize("x_type", ref.TYPES)
@pytest.mark.parametrize("out_type", ref.TYPES)
@pytest.mark.parametrize("dim,rot", [(128, 128), (72, 36)])
def test_rope_types(cuda, x_type, out_type, dim, rot):
    from tacker_b200 import ops

    heads, kv_heads, tokens = 4, 2, 33
    width = (heads + 2 * kv_heads) * dim
    x, bias = normal(cuda, 1, tokens, width, type=x_type), normal(cuda, 2, width)
    turns = cuda.tensor(ops.rope_turns(rot)[0], dtype=cuda.float64, device="cuda")
    pos = cuda.arange(tokens, dtype=cuda.int32, device="cuda") * 1001
    q, k, v = (cuda.zeros(tokens, h, dim, dtype=ref.TYPES[out_type], device="cuda") for h in (heads, kv_heads, kv_heads))
    ops.rope_qkv(at(x), ref.CODES[x_type], width, at(bias), at(pos), at(turns), rot, 0, 1.1, tokens, heads, kv_heads, dim, at(q), heads * dim,
                 at(k), kv_heads * dim, at(v), kv_heads * dim, ref.CODES[out_type])
    cuda.cuda.synchronize()
    want, tol = ref.rope(x, bias, pos, turns, rot, 0, 1.1, heads, kv_heads, dim, out_type)
    within(cuda, cuda.cat((q, k, v), 1), want, tol, "heads")


# ---- a block of them -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("q_len,past", [([100, 3, 37, 1], [0, 0, 0, 0]), ([1] * 9, [0, 5, 17, 63, 64, 200, 255, 100, 31])])
def test_block_first_norm_and_its_rows_in_8_bits(cuda, q_len, past):
    """The first norm's result, which the block's last norm overwrites, and its rounding to 8 bits."""
    from tacker_b200 import ops

    b = Block(cuda, q_len, past)
    b.run()
    h = cuda.zeros_like(b.h)
    ops.norm_residual_rows(at(b.branch), 0, b.cols, 0, 0, 0, 0, 0, 1, 1.0, at(b.stream), b.cols, 0, 0, 0, at(b.gamma[0]), 0, at(h), b.cols, 2, 0,
                           1e-6, b.T, b.cols)
    cuda.cuda.synchronize()
    _, want, _, tol = ref.norm(b.branch, b.stream, None, 1, 1.0, 0, None, None, b.gamma[0], None, 0, 1e-6, "f32", "bf16")
    within(cuda, h, want, tol, "input of the projection")
    codes, scales = ref.quantize(h)
    assert cuda.equal(codes, b.c1.double()) and cuda.equal(scales, b.r1)


def test_two_host_threads(cuda):
    """Blocks of different shapes issued by two threads at once, each on a stream of its own: what each gives alone."""
    import threading

    blocks = [Block(cuda, [1] * 7, [3, 64, 200, 7, 0, 31, 90]), Block(cuda, [100, 3, 37, 80], [0, 20, 0, 5], dim=128)]
    alone = []
    for b in blocks:
        b.run()
        cuda.cuda.synchronize()
        alone.append(b.outputs())
    streams, errors, gate = [cuda.cuda.Stream() for _ in blocks], [], threading.Barrier(2)

    def issue(b, s):
        try:
            gate.wait(30)
            for _ in range(50):
                b.run(s.cuda_stream)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=issue, args=x) for x in zip(blocks, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and not any(t.is_alive() for t in threads)
    cuda.cuda.synchronize()
    for b, want in zip(blocks, alone):
        for x, y in zip(b.outputs(), want):
            assert cuda.equal(x, y)


def test_no_wait_ran_out(cuda):
    from tacker_b200 import ops

    assert ops.device_status() == 0
