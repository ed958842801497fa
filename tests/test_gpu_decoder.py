"""The decoder-block operators against their definitions in binary64 (B200 only)."""
import math
import random

import pytest

import decoder_ref as ref

pytestmark = pytest.mark.gpu


def normal(torch, seed, *shape, type="f32", scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(ref.TYPES[type])


def at(x):
    return 0 if x is None else x.data_ptr()


def within(torch, got, want, tol, what):
    """got within tol of want, infinities equal, and no NaN where there is none to have."""
    got = got.double()
    same = (got == want) | ((got - want).abs() <= tol)
    assert bool(same.all()), f"{what}: {int((~same).sum())} of {same.numel()} off, first at {(~same).nonzero()[0].tolist()}: " \
        f"{got[~same][0].item()} for {want[~same][0].item()} +- {tol[~same][0].item() if tol.shape == same.shape else tol}"


# ---- attention -----------------------------------------------------------------------------------------------------
class Attention:
    """One call over packed sequences, checked in full: outputs, lse, rows that belong to no sequence, unused cache rows."""

    def __init__(self, torch, q_len, k_len, heads, kv_heads, dim, type, causal, *, slab=0, lead=0, behind=0, pad=0, seed=1,
                 shift=0, scale=None, poison=True):
        self.torch, self.q_len, self.k_len = torch, q_len, k_len
        self.heads, self.kv_heads, self.dim, self.type, self.causal = heads, kv_heads, dim, type, causal
        n = len(q_len)
        self.q_start = [lead + sum(q_len[:i]) for i in range(n + 1)]
        self.total = self.q_start[-1] + behind
        self.k_start = [slab * i for i in range(n)] if slab else [shift + sum(k_len[:i]) for i in range(n)]
        self.rows = max([1] + [slab * n if slab else shift + sum(k_len) + shift])
        self.scale = 1 / math.sqrt(dim) if scale is None else scale
        make = lambda s, r, h: normal(torch, s, r, h * dim + pad, type=type)[:, :h * dim].unflatten(1, (h, dim))  # noqa: E731
        self.q, self.k, self.v = make(seed, max(self.total, 1), heads), make(seed + 1, self.rows, kv_heads), make(seed + 2, self.rows, kv_heads)
        if poison:  # what no sequence owns may hold anything
            used = torch.zeros(self.rows, dtype=torch.bool, device="cuda")
            for s, m in zip(self.k_start, k_len):
                used[s:s + m] = True
            self.k[~used], self.v[~used] = math.nan, math.inf
        self.out = torch.full((max(self.total, 1), heads * dim + pad), 7.0, dtype=ref.TYPES[type], device="cuda")
        self.lse = torch.full((max(self.total, 1), heads), 7.0, device="cuda")
        self.index = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (self.q_start, self.k_start, self.k_len)]
        self.pad = pad

    def call(self, workspace=None, stream=0, max_q=None, max_k=None, lse=True):
        from tacker_b200 import ops

        d, pad = self.dim, self.pad
        ops.attention_packed(at(self.q), self.heads * d + pad, at(self.k), self.kv_heads * d + pad, at(self.v),
                             self.kv_heads * d + pad, at(self.out), self.heads * d + pad, at(self.lse) if lse else 0,
                             ref.CODES[self.type], *(at(x) for x in self.index), len(self.q_len), self.total, self.rows,
                             max(self.q_len) if max_q is None else max_q, max(self.k_len) if max_k is None else max_k,
                             self.heads, self.kv_heads, d, self.scale, self.causal, at(workspace),
                             0 if workspace is None else workspace.numel(), stream=stream)
        return self

    def check(self, lse=True):
        torch = self.torch
        torch.cuda.synchronize()
        want, want_lse, tol, tol_lse = ref.attention(self.q, self.k, self.v, self.q_start, self.k_start, self.k_len,
                                                     self.scale, self.causal, self.type)
        got = self.out[:, :self.heads * self.dim].unflatten(1, (self.heads, self.dim))
        a, b = self.q_start[0], self.q_start[-1]
        within(torch, got[a:b], want[a:b], tol[a:b], "out")
        if lse:
            within(torch, self.lse[a:b], want_lse[a:b], tol_lse[a:b], "lse")
        else:
            assert bool((self.lse == 7).all())
        for rest in (got[:a], got[b:], self.lse[:a], self.lse[b:], self.out[:, self.heads * self.dim:]):
            assert bool((rest == 7).all()), "wrote outside the sequences' rows"


def workspace(torch, size=64 << 20):
    return torch.empty(size, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (8, 2), (7, 1), (15, 3), (16, 1)])
def test_attention_prompts(cuda, type, dim, causal, heads, kv_heads):
    """Packed prompts of one token to several tiles, lengths on both sides of every tile border."""
    lens = [1, 2, 17, 64, 127, 128, 129, 255, 256, 257, 300]
    Attention(cuda, lens, lens, heads, kv_heads, dim, type, causal).call(workspace(cuda)).check()


@pytest.mark.parametrize("dim", [8, 40, 72, 80, 96, 100, 120, 160, 256])
def test_attention_head_sizes(cuda, dim):
    lens = [3, 130, 65]
    Attention(cuda, lens, lens, 6, 2, dim, "f16", True).call(workspace(cuda)).check()
    Attention(cuda, [1, 1, 1], [3, 700, 65], 6, 2, dim, "bf16", True, slab=701).call(workspace(cuda)).check()


@pytest.mark.parametrize("causal", [True, False])
def test_attention_chunks_behind_a_cache(cuda, causal):
    """More keys than queries, fewer keys than queries (the first rows then see nothing), no keys, no queries."""
    q_len, k_len = [5, 130, 0, 64, 33, 1, 200], [133, 1000, 50, 40, 0, 0, 200]
    Attention(cuda, q_len, k_len, 8, 2, 128, "bf16", causal, slab=1024, lead=3, behind=5).call(workspace(cuda)).check()
    Attention(cuda, q_len, k_len, 8, 2, 64, "f16", causal, lead=3, behind=5, shift=7, pad=8).call(workspace(cuda)).check()


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(12, 12), (32, 8), (7, 1), (16, 1), (40, 1), (64, 2)])
def test_attention_single_tokens(cuda, type, dim, heads, kv_heads):
    rng = random.Random(heads * dim)
    k_len = [1, 2, 15, 16, 17, 63, 64, 65, 0, 128, 1500] + [rng.randint(1, 600) for _ in range(4)]
    for ws in (workspace(cuda), None, workspace(cuda, 100_000)):
        Attention(cuda, [1] * len(k_len), k_len, heads, kv_heads, dim, type, True, slab=1501).call(ws).check()


@pytest.mark.parametrize("q", [2, 3, 5, 9])
def test_attention_a_few_tokens_each(cuda, q):
    k_len = [q, 700, 3, 1200]
    Attention(cuda, [q, 1, q, q - 1], k_len, 8, 2, 128, "f16", True, slab=1200).call(workspace(cuda)).check()


def test_attention_long_axis(cuda):
    """Two tokens over long caches: the key axis is split; and the same without room to split."""
    a = Attention(cuda, [1, 1], [40001, 33333], 16, 2, 128, "f16", True, slab=40010)
    a.call(workspace(cuda)).check()
    a.out.fill_(7)
    a.call().check()


@pytest.mark.parametrize("max_q,max_k", [(1, 1), (4096, 100000), (0, 0)])
def test_attention_bounds_are_hints(cuda, max_q, max_k):
    """max_q and max_k choose the launch, not the result."""
    Attention(cuda, [1, 40, 300], [500, 40, 310], 8, 2, 64, "bf16", True, slab=600).call(workspace(cuda), max_q=max_q, max_k=max_k).check()


def test_attention_sharp_and_flat_scores(cuda):
    """Scores that rise along the keys by far more than the largest weight holds, and scores that are all equal."""
    a = Attention(cuda, [300, 1], [300, 900], 4, 2, 128, "f16", True, scale=1.0, slab=900)
    a.k.mul_(cuda.linspace(0.1, 4, a.rows, device="cuda")[:, None, None].half())
    a.call(workspace(cuda)).check()
    a = Attention(cuda, [300, 1], [300, 900], 4, 2, 64, "bf16", False, scale=0.0)
    a.call(workspace(cuda)).check()
    a = Attention(cuda, [200, 1], [200, 900], 4, 2, 64, "bf16", True, scale=-0.3)
    a.call(workspace(cuda)).check()


def test_attention_without_lse_and_unaligned(cuda):
    lens = [70, 1, 9]
    Attention(cuda, lens, lens, 4, 2, 64, "f16", True).call(workspace(cuda), lse=False).check(lse=False)
    a = Attention(cuda, lens, lens, 4, 2, 64, "f16", True, pad=1)  # rows that start on odd addresses
    a.call(workspace(cuda)).check()


def test_attention_keys_beyond_the_diagonal_do_not_reach_a_query(cuda):
    """Keys that the mask hides may score anything (their values are finite)."""
    a = Attention(cuda, [200], [200], 4, 2, 128, "f16", True)
    a.call(workspace(cuda))
    cuda.cuda.synchronize()
    first = a.out.clone()
    a.k[150:] = math.nan
    a.call(workspace(cuda))
    cuda.cuda.synchronize()
    assert cuda.equal(first[:150], a.out[:150])
    assert bool(a.out[150:].isnan().all())


def test_attention_bad_index_arrays_stay_inside_the_tensors(cuda):
    """Starts and lengths outside the tensors: clamped to them; nothing is read or written elsewhere."""
    a = Attention(cuda, [4, 4], [4, 4], 4, 2, 64, "f16", True, lead=2, behind=2, slab=8)
    a.index[1].copy_(cuda.tensor([-5, 1 << 30], dtype=cuda.int32))
    a.index[2].copy_(cuda.tensor([1 << 30, 1 << 30], dtype=cuda.int32))
    a.call(workspace(cuda))
    cuda.cuda.synchronize()
    assert bool((a.out[2:10] == 0).all()) and bool((a.lse[2:10] == -math.inf).all())
    a.index[0].copy_(cuda.tensor([-3, 100, 7], dtype=cuda.int32))
    a.call(workspace(cuda))
    cuda.cuda.synchronize()


@pytest.mark.parametrize("causal", [True, False])
def test_attention_more_items_than_sms(cuda, causal):
    """Several hundred work items of very different lengths: every CTA takes over blocks that have not started."""
    lens = [2500, 3, 1700, 129, 700]
    Attention(cuda, lens, lens, 16, 16, 64, "f16", causal).call().check()
    Attention(cuda, lens[1:], [n + 500 for n in lens[1:]], 24, 8, 128, "bf16", causal).call().check()


@pytest.mark.parametrize("heads,kv_heads", [(128, 1), (65, 1), (130, 1), (96, 2)])
def test_attention_large_groups(cuda, heads, kv_heads):
    """Groups of a whole tile, of half a tile and one more, and larger than a tile."""
    Attention(cuda, [1, 40, 3], [700, 40, 133], heads, kv_heads, 64, "f16", True).call(workspace(cuda)).check()


def test_attention_shared_keys(cuda):
    """Sequences that read the same rows of the cache (a common prefix), and one that reads them behind others."""
    for q_len in ([1, 1, 1], [130, 70, 5]):
        a = Attention(cuda, q_len, [300, 200, 250], 8, 2, 128, "bf16", True, slab=300, poison=False)
        a.k_start = [0, 0, 50]
        a.index[1].copy_(cuda.tensor(a.k_start, dtype=cuda.int32))
        a.call(workspace(cuda)).check()


def test_attention_offsets_beyond_32_bits(cuda):
    """A cache of more than 2^31 elements whose last rows are the ones in use; new keys written there by slots."""
    from tacker_b200 import ops

    kv_heads, dim, rows = 8, 128, 2_100_100
    for q_len in ([1, 1], [100, 33]):
        a = Attention(cuda, q_len, [700, 320], 16, kv_heads, dim, "bf16", True, poison=False)
        k, v = (cuda.empty(rows, kv_heads, dim, dtype=cuda.bfloat16, device="cuda") for _ in "kv")
        a.k_start = [rows - 1100, rows - 320]
        for s, n in zip(a.k_start, a.k_len):
            k[s:s + n], v[s:s + n] = normal(cuda, s, n, kv_heads, dim, type="bf16"), normal(cuda, s + 1, n, kv_heads, dim, type="bf16")
        a.k, a.v, a.rows = k, v, rows
        a.index[1].copy_(cuda.tensor(a.k_start, dtype=cuda.int32))
        a.call(workspace(cuda)).check()
    x = normal(cuda, 5, 2, (2 + 2 * kv_heads) * dim)
    q, slots, pos = cuda.zeros(2, 2, dim, dtype=cuda.bfloat16, device="cuda"), cuda.tensor([rows - 1, rows - 7], device="cuda"), cuda.zeros(2, dtype=cuda.int32, device="cuda")
    turns = cuda.zeros(1, dtype=cuda.float64, device="cuda")
    ops.rope_qkv(at(x), 0, x.shape[1], 0, at(pos), at(turns), 2, 0, 1.0, 2, 2, kv_heads, dim, at(q), 2 * dim, at(k), kv_heads * dim, at(v),
                 kv_heads * dim, 2, at(slots), rows)
    cuda.cuda.synchronize()
    heads = x.view(2, -1, dim).bfloat16()
    assert cuda.equal(k[slots], heads[:, 2:2 + kv_heads]) and cuda.equal(v[slots], heads[:, 2 + kv_heads:])


# ---- rotary heads --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("x_type,out_type", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (80, 32), (96, 0), (64, 20), (72, 72), (6, 4), (256, 256)])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_rope(cuda, x_type, out_type, dim, rot, interleaved):
    from tacker_b200 import ops

    heads, kv_heads, tokens, width = 6, 2, 13, 10 * dim
    x, bias = normal(cuda, 1, tokens, width, type=x_type), normal(cuda, 2, width)
    turns, magnitude = ops.rope_turns(rot, 10000.0, ops.ROPE_RAMP, 8.0, 4096.0) if rot else ([0.0], 1.0)
    turns = cuda.tensor(turns, dtype=cuda.float64, device="cuda")
    pos = cuda.tensor([0, 1, 2, 7, 1000, 4095, 65537, 999_999, 2_000_003, 2**31 - 1, 5, 5, -3], dtype=cuda.int32, device="cuda")
    slots = cuda.tensor([3, 0, -1, 19, 7, 20, 1 << 40, 2, 4, 5, 6, 9, 8], dtype=cuda.int64, device="cuda")
    for b, sl in ((bias, slots), (None, None)):
        rows = 20 if sl is not None else tokens
        q, k, v = (cuda.full((r, h, dim), 7.0, dtype=ref.TYPES[out_type], device="cuda") for r, h in ((tokens, heads), (rows, kv_heads), (rows, kv_heads)))
        ops.rope_qkv(at(x), ref.CODES[x_type], width, at(b), at(pos), at(turns), rot, interleaved, magnitude, tokens, heads,
                     kv_heads, dim, at(q), heads * dim, at(k), kv_heads * dim, at(v), kv_heads * dim, ref.CODES[out_type],
                     at(sl), rows if sl is not None else 0)
        cuda.cuda.synchronize()
        want, tol = ref.rope(x, b, pos, turns[:rot // 2], rot, interleaved, magnitude, heads, kv_heads, dim, out_type)
        within(cuda, q, want[:, :heads], tol[:, :heads], "q")
        where = list(range(tokens)) if sl is None else [s if 0 <= s < rows else None for s in sl.tolist()]
        for t, r in enumerate(where):
            if r is not None:
                within(cuda, k[r], want[t, heads:heads + kv_heads], tol[t, heads:heads + kv_heads], "k")
                within(cuda, v[r], want[t, heads + kv_heads:], tol[t, heads + kv_heads:], "v")
        for r in set(range(rows)) - set(where):
            assert bool((k[r] == 7).all()) and bool((v[r] == 7).all()), "wrote a row that no slot names"


def test_rope_strides_and_many_tokens(cuda):
    """Leading dimensions beyond the heads, q, k and v inside wider rows, and unaligned starts."""
    from tacker_b200 import ops

    heads, kv_heads, dim, rot, tokens = 12, 4, 64, 64, 700
    width = (heads + 2 * kv_heads) * dim
    turns = cuda.tensor(ops.rope_turns(rot)[0], dtype=cuda.float64, device="cuda")
    pos = cuda.arange(tokens, dtype=cuda.int32, device="cuda")
    for extra, off in ((8, 0), (8, 1), (3, 0)):
        x = normal(cuda, 3, tokens * (width + extra) + 8)[off:off + tokens * (width + extra)].view(tokens, width + extra)
        big = cuda.full((tokens, width + extra), 7.0, dtype=cuda.bfloat16, device="cuda")
        q, k, v = big[:, :heads * dim], big[:, heads * dim:(heads + kv_heads) * dim], big[:, (heads + kv_heads) * dim:width]
        ops.rope_qkv(at(x), 0, width + extra, 0, at(pos), at(turns), rot, 0, 1.0, tokens, heads, kv_heads, dim, at(q),
                     width + extra, at(k), width + extra, at(v), width + extra, 2)
        cuda.cuda.synchronize()
        want, tol = ref.rope(x[:, :width], None, pos, turns, rot, 0, 1.0, heads, kv_heads, dim, "bf16")
        within(cuda, big[:, :width].view(tokens, -1, dim), want, tol, "heads")
        assert bool((big[:, width:] == 7).all())


# ---- the residual stream -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layer", [0, 1])
@pytest.mark.parametrize("post", [0, 1])
@pytest.mark.parametrize("types", [("f32", "f32", "f16"), ("bf16", "bf16", "bf16"), ("f16", "f32", "f32"), ("f32", "bf16", "f16")])
@pytest.mark.parametrize("rows,cols,gate_rows", [(1, 8, 0), (5, 59, 2), (37, 768, 16), (9, 4096, 1), (3, 8192, 0), (130, 264, 128), (2, 40000, 0)])
def test_norm(cuda, layer, post, types, rows, cols, gate_rows):
    from tacker_b200 import ops

    a_type, x_type, h_type = types
    a, x = normal(cuda, 1, rows, cols, type=a_type, scale=3), normal(cuda, 2, rows, cols, type=x_type, scale=2)
    gs = [1 + normal(cuda, 3 + i, cols, scale=0.2) for i in range(4)]
    gate = normal(cuda, 9, -(-rows // gate_rows), cols) if gate_rows else None
    y, h = cuda.zeros(rows, cols, dtype=ref.TYPES[x_type], device="cuda"), cuda.zeros(rows, cols, dtype=ref.TYPES[h_type], device="cuda")
    args = dict(scale=0.3, post=post, layer=layer, eps=1e-5)

    def call(x, y, h, g):
        ops.norm_residual_rows(at(a), ref.CODES[a_type], cols, post, at(g[0]), at(g[1]), at(gate), cols, max(gate_rows, 1), 0.3,
                               at(x), cols, at(y), cols, ref.CODES[x_type], at(g[2]), at(g[3]), at(h), cols,
                               ref.CODES[h_type], layer, 1e-5, rows, cols)
        cuda.cuda.synchronize()

    def want(x, g):
        return ref.norm(a, x, gate, max(gate_rows, 1), post_gamma=g[0], post_beta=g[1], pre_gamma=g[2], pre_beta=g[3],
                        x_type=x_type, h_type=h_type, **args)

    for g, stream in ((gs, x), ([None] * 4, None)):
        wy, wh, ty, th = want(stream, g)
        call(stream, y, h, g)
        within(cuda, y, wy, ty, "y")
        within(cuda, h, wh, th, "h")
    wy, wh, ty, th = want(x, gs)
    only = cuda.full_like(y, 7.0)
    call(x, only, None, gs)
    within(cuda, only, wy, ty, "y alone")
    call(x, None, h, gs)
    within(cuda, h, wh, th, "h alone")
    call(x, x, h, gs)  # the residual stream in place
    within(cuda, x, wy, ty, "y in place")
    within(cuda, h, wh, th, "h of y in place")


def test_norm_strides_and_constant_rows(cuda):
    """Rows inside wider arrays, and rows without spread: a layer norm of a constant is its beta, a norm of zeros zero."""
    from tacker_b200 import ops

    rows, cols, ld = 33, 640, 704
    a, x = normal(cuda, 1, rows, ld, type="bf16"), normal(cuda, 2, rows, ld)
    y, h = cuda.full((rows, ld), 7.0, device="cuda"), cuda.full((rows, ld), 7.0, dtype=cuda.float16, device="cuda")
    ops.norm_residual_rows(at(a), 2, ld, 1, 0, 0, 0, 0, 1, 1.0, at(x), ld, at(y), ld, 0, 0, 0, at(h), ld, 1, 0, 1e-6, rows, cols)
    cuda.cuda.synchronize()
    wy, wh, ty, th = ref.norm(a[:, :cols], x[:, :cols], None, 1, 1.0, 1, None, None, None, None, 0, 1e-6, "f32", "f16")
    within(cuda, y[:, :cols], wy, ty, "y")
    within(cuda, h[:, :cols], wh, th, "h")
    assert bool((y[:, cols:] == 7).all()) and bool((h[:, cols:] == 7).all())
    zero, beta = cuda.zeros(rows, cols, device="cuda"), normal(cuda, 4, cols)
    five = cuda.full((rows, cols), 5.0, device="cuda")
    for src, want in ((zero, beta), (five, beta)):
        ops.norm_residual_rows(at(src), 0, cols, 0, 0, 0, 0, 0, 1, 1.0, 0, 0, 0, 0, 0, 0, at(beta), at(h), cols, 1, 1, 1e-6, rows, cols)
        cuda.cuda.synchronize()
        assert cuda.equal(h.flatten()[:rows * cols].view(rows, cols), want.half().expand(rows, cols))


# ---- 8-bit rows and products ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (64, 4096), (17, 1000), (130, 8), (2, 70000)])
def test_quantize(cuda, type, rows, cols):
    from tacker_b200 import ops

    x = normal(cuda, rows + cols, rows, cols, type=type, scale=2)
    if rows > 2:
        x[1] = 0
        x[2, 0] = x[2].abs().max()
        x[2, 1:] = x[2, 0] * (cuda.arange(cols - 1, device="cuda") % 255 - 127).to(x.dtype) / 254  # halves of a step
    codes, scales = cuda.full((rows, cols), 9, dtype=cuda.int8, device="cuda"), cuda.zeros(rows, device="cuda")
    ops.quantize_rows_i8(at(x), ref.CODES[type], cols, at(codes), cols, at(scales), rows, cols)
    cuda.cuda.synchronize()
    want, ws = ref.quantize(x)
    assert cuda.equal(scales, ws)
    assert cuda.equal(codes.double(), want)


def test_quantize_halves_of_the_largest(cuda):
    """x = (j + 1/2) / 127 of the largest, for largest values of every mantissa a short type has: all borders there are."""
    from tacker_b200 import ops

    top = cuda.arange(1024, 2048, device="cuda").half()
    x = (top.double()[:, None] * (cuda.arange(254, device="cuda") + 0.5)[None] / 254).half()
    x = cuda.cat((x, -x, top[:, None], top[:, None] / 2), 1).contiguous()
    rows, cols = x.shape
    codes, scales = cuda.zeros(rows, cols, dtype=cuda.int8, device="cuda"), cuda.zeros(rows, device="cuda")
    ops.quantize_rows_i8(at(x), 1, cols, at(codes), cols, at(scales), rows, cols)
    cuda.cuda.synchronize()
    want, ws = ref.quantize(x)
    assert cuda.equal(scales, ws) and cuda.equal(codes.double(), want)


def test_quantize_rows_that_have_no_scale(cuda):
    from tacker_b200 import ops

    x = normal(cuda, 1, 5, 64)
    x[1, 3], x[2, 63], x[3], x[4] = math.nan, -math.inf, x[3] * 1e-37, x[4] * 1e-40
    codes, scales = cuda.full((5, 72), 9, dtype=cuda.int8, device="cuda"), cuda.zeros(5, device="cuda")
    ops.quantize_rows_i8(at(x), 0, 64, at(codes), 72, at(scales), 5, 64)
    cuda.cuda.synchronize()
    assert math.isnan(scales[1].item()) and scales[2].item() == math.inf and scales[4].item() == 0
    assert not codes[1:3, :64].any() and not codes[4, :64].any() and bool((codes[:, 64:] == 9).all())
    for r in (0, 3):
        want, ws = ref.quantize(x[r:r + 1])
        assert cuda.equal(scales[r:r + 1], ws) and cuda.equal(codes[r:r + 1, :64].double(), want)


@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 128, 128), (3, 333, 48), (16, 4096, 4096), (17, 130, 2048), (33, 1000, 1040),
                                   (64, 512, 16384), (65, 64, 128), (127, 129, 130), (128, 256, 512), (130, 1234, 1040),
                                   (300, 77, 4096), (1001, 515, 640), (512, 768, 100), (2048, 2048, 256),
                                   (1537, 2305, 200), (2304, 1280, 1040), (70, 12000, 64), (1030, 8200, 16)])
def test_i8gemm(cuda, out_type, M, N, K):
    from tacker_b200 import ops

    ld = -(-K // 16) * 16 + (16 if M % 2 else 0)
    g = cuda.Generator(device="cuda")
    g.manual_seed(M + N + K)
    a, b = (cuda.randint(-128, 128, (r, ld), generator=g, device="cuda", dtype=cuda.int8) for r in (M, N))
    sa, sb, bias = normal(cuda, 1, M).abs() / 100, normal(cuda, 2, N).abs() / 100, normal(cuda, 3, N)
    pad = N % 3
    for bb in (bias, None):
        out = cuda.full((M, N + pad), 7.0, dtype=ref.TYPES[out_type], device="cuda")
        ops.i8gemm(at(a), ld, at(sa), at(b), ld, at(sb), at(bb), at(out), N + pad, ref.CODES[out_type], M, N, K)
        cuda.cuda.synchronize()
        want, tol = ref.i8gemm(a[:, :K], sa, b[:, :K], sb, bb, out_type)
        within(cuda, out[:, :N], want, tol, "out")
        assert bool((out[:, N:] == 7).all())


@pytest.mark.parametrize("M,N", [(2, 128), (128, 128), (600, 512)])
def test_i8gemm_largest_sums(cuda, M, N):
    """The longest k with every product at its largest: 131071 * 2^14 is the last sum that fits."""
    from tacker_b200 import ops

    K, ld = 131071, 131072
    a, b = (cuda.full((r, ld), -128, dtype=cuda.int8, device="cuda") for r in (M, N))
    a[1] = 127
    out, one = cuda.zeros(M, N, device="cuda"), cuda.ones(max(M, N), device="cuda")
    ops.i8gemm(at(a), ld, at(one), at(b), ld, at(one), 0, at(out), N, 0, M, N, K)
    cuda.cuda.synchronize()
    want = cuda.full((M, N), float(K * 16384), device="cuda")
    want[1] = float(-K * 127 * 128)
    assert cuda.equal(out, want)


# ---- a block of them -----------------------------------------------------------------------------------------------
class Block:
    """norm -> rows to 8 bits -> fused projection -> rotary heads into a cache -> attention -> rows to 8 bits -> output
    projection -> norm behind it into the residual stream, over packed tokens."""

    def __init__(self, torch, q_len, past, heads=8, kv_heads=2, dim=64, cols=512, slab=256):
        from tacker_b200 import ops

        self.torch, self.q_len, self.past = torch, q_len, past
        self.heads, self.kv_heads, self.dim, self.cols, self.slab = heads, kv_heads, dim, cols, slab
        self.T, n = sum(q_len), len(q_len)
        width = (heads + 2 * kv_heads) * dim
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.index = [i32([sum(q_len[:i]) for i in range(n + 1)]), i32([slab * i for i in range(n)]),
                      i32([p + q for p, q in zip(past, q_len)])]
        self.pos = i32([p + t for p, q in zip(past, q_len) for t in range(q)])
        self.slots = torch.tensor([slab * i + p + t for i, (p, q) in enumerate(zip(past, q_len)) for t in range(q)], device="cuda")
        self.turns = torch.tensor(ops.rope_turns(dim)[0], dtype=torch.float64, device="cuda")
        self.stream = normal(torch, 1, self.T, cols)
        self.branch = normal(torch, 2, self.T, cols)
        self.gamma = [1 + normal(torch, 3 + i, cols, scale=0.1) for i in range(3)]
        self.w1, self.s1 = (t.contiguous() for t in ref.quantize(normal(torch, 7, width, cols, scale=cols ** -0.5)))
        self.w2, self.s2 = (t.contiguous() for t in ref.quantize(normal(torch, 8, cols, heads * dim, scale=(heads * dim) ** -0.5)))
        self.w1, self.w2 = self.w1.to(torch.int8), self.w2.to(torch.int8)
        self.k, self.v = (normal(torch, s, slab * n, kv_heads, dim, type="bf16") for s in (9, 10))
        z = lambda *s, t="bf16": torch.zeros(*s, dtype=ref.TYPES[t], device="cuda")  # noqa: E731
        self.y, self.h, self.c1, self.r1 = z(self.T, cols, t="f32"), z(self.T, cols), z(self.T, cols).to(torch.int8), z(self.T, t="f32")
        self.qkv, self.q, self.o = z(self.T, width, t="f32"), z(self.T, heads, dim), z(self.T, heads, dim)
        self.c2, self.r2, self.p, self.y2 = z(self.T, heads * dim).to(torch.int8), z(self.T, t="f32"), z(self.T, cols, t="f32"), z(self.T, cols, t="f32")
        self.ws = workspace(torch, 8 << 20)

    def run(self, stream=0):
        from tacker_b200 import ops

        T, c, h, hk, d, n = self.T, self.cols, self.heads, self.kv_heads, self.dim, len(self.q_len)
        w = (h + 2 * hk) * d
        ops.norm_residual_rows(at(self.branch), 0, c, 0, 0, 0, 0, 0, 1, 1.0, at(self.stream), c, at(self.y), c, 0,
                               at(self.gamma[0]), 0, at(self.h), c, 2, 0, 1e-6, T, c, stream=stream)
        ops.quantize_rows_i8(at(self.h), 2, c, at(self.c1), c, at(self.r1), T, c, stream=stream)
        ops.i8gemm(at(self.c1), c, at(self.r1), at(self.w1), c, at(self.s1), 0, at(self.qkv), w, 0, T, w, c, stream=stream)
        ops.rope_qkv(at(self.qkv), 0, w, 0, at(self.pos), at(self.turns), d, 0, 1.0, T, h, hk, d, at(self.q), h * d, at(self.k),
                     hk * d, at(self.v), hk * d, 2, at(self.slots), self.k.shape[0], stream=stream)
        ops.attention_packed(at(self.q), h * d, at(self.k), hk * d, at(self.v), hk * d, at(self.o), h * d, 0, 2,
                             *(at(x) for x in self.index), n, T, self.k.shape[0], max(self.q_len), self.slab, h, hk, d,
                             d ** -0.5, 1, at(self.ws), self.ws.numel(), stream=stream)
        ops.quantize_rows_i8(at(self.o), 2, h * d, at(self.c2), h * d, at(self.r2), T, h * d, stream=stream)
        ops.i8gemm(at(self.c2), h * d, at(self.r2), at(self.w2), h * d, at(self.s2), 0, at(self.p), c, 0, T, c, h * d, stream=stream)
        ops.norm_residual_rows(at(self.p), 0, c, 1, at(self.gamma[1]), 0, 0, 0, 1, 0.5, at(self.y), c, at(self.y2), c, 0,
                               at(self.gamma[2]), 0, at(self.h), c, 2, 0, 1e-6, T, c, stream=stream)

    def outputs(self):
        return [x.clone() for x in (self.y, self.c1, self.r1, self.qkv, self.q, self.k, self.v, self.o, self.c2, self.r2, self.p, self.y2, self.h)]

    def check(self):
        torch, h, hk, d = self.torch, self.heads, self.kv_heads, self.dim
        torch.cuda.synchronize()
        y, _, ty, _ = ref.norm(self.branch, self.stream, None, 1, 1.0, 0, None, None, self.gamma[0], None, 0, 1e-6, "f32", "bf16")
        within(torch, self.y, y, ty, "residual stream")
        want, tol = ref.i8gemm(self.c1, self.r1, self.w1, self.s1, None, "f32")
        within(torch, self.qkv, want, tol, "projection")
        want, tol = ref.rope(self.qkv, None, self.pos, self.turns, d, 0, 1.0, h, hk, d, "bf16")
        within(torch, self.q, want[:, :h], tol[:, :h], "query heads")
        within(torch, self.k[self.slots], want[:, h:h + hk], tol[:, h:h + hk], "keys in the cache")
        within(torch, self.v[self.slots], want[:, h + hk:], tol[:, h + hk:], "values in the cache")
        q0, k0, kl = (x.tolist() for x in self.index)
        want, _, tol, _ = ref.attention(self.q, self.k, self.v, q0, k0, kl, d ** -0.5, True, "bf16")
        within(torch, self.o, want, tol, "context")
        codes, scales = ref.quantize(self.o.flatten(1))
        assert torch.equal(codes, self.c2.double()) and torch.equal(scales, self.r2)
        want, tol = ref.i8gemm(self.c2, self.r2, self.w2, self.s2, None, "f32")
        within(torch, self.p, want, tol, "output projection")
        y2, hh, ty, th = ref.norm(self.p, self.y, None, 1, 0.5, 1, self.gamma[1], None, self.gamma[2], None, 0, 1e-6, "f32", "bf16")
        within(torch, self.y2, y2, ty, "residual stream behind the block")
        within(torch, self.h, hh, th, "next block's input")


@pytest.mark.parametrize("q_len,past", [([100, 3, 37, 1], [0, 0, 0, 0]), ([1] * 9, [0, 5, 17, 63, 64, 200, 255, 100, 31]),
                                        ([20, 1, 64], [100, 90, 0])])
def test_block(cuda, q_len, past):
    b = Block(cuda, q_len, past)
    b.run()
    b.check()


def test_block_captured_and_replayed(cuda):
    """On a stream of its own and inside a graph, with new inputs and other lengths in the same buffers: bit for bit what
    plain calls give."""
    b = Block(cuda, [1] * 5, [3, 64, 200, 7, 0])
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    with cuda.cuda.stream(side):
        b.run(side.cuda_stream)
    side.synchronize()
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph, stream=side):
        b.run(cuda.cuda.current_stream().cuda_stream)
    for seed in (21, 22):
        b.stream.copy_(normal(cuda, seed, b.T, b.cols))
        b.index[2].add_(1)
        b.pos.add_(1)
        b.slots.add_(1)
        cuda.cuda.synchronize()
        graph.replay()
        cuda.cuda.synchronize()
        got = b.outputs()
        b.run()
        cuda.cuda.synchronize()
        for x, y in zip(got, b.outputs()):
            assert cuda.equal(x, y)
        b.check()


def test_two_streams_at_once(cuda):
    """Blocks of single tokens and of prompts on two streams with buffers of their own, over and over: each gives what it
    gives alone."""
    blocks = [Block(cuda, [1] * 7, [3, 64, 200, 7, 0, 31, 90]), Block(cuda, [100, 3, 37, 80], [0, 20, 0, 5])]
    alone = []
    for b in blocks:
        b.run()
        cuda.cuda.synchronize()
        alone.append(b.outputs())
    streams = [cuda.cuda.Stream() for _ in blocks]
    for _ in range(20):
        for b, s in zip(blocks, streams):
            b.run(s.cuda_stream)
    cuda.cuda.synchronize()
    for b, want in zip(blocks, alone):
        for x, y in zip(b.outputs(), want):
            assert cuda.equal(x, y)


def test_no_wait_ran_out(cuda):
    from tacker_b200 import ops

    assert ops.device_status() == 0
