"""What the decoder-block entry points refuse, and the rotary plan (no GPU needed)."""
import math

import pytest

P = 1 << 20  # an aligned address that is never touched: the calls end at their checks
ARGS, ALIGN, SHAPE = -1, -2, -3


@pytest.fixture(scope="module")
def ops():
    from tacker_b200 import _build, ops

    _build.build_library()
    return ops


def refused(status, call, *args, **kw):
    import tacker_b200

    with pytest.raises(tacker_b200.TackerError) as e:
        call(*args, **kw)
    assert e.value.status == status, (e.value.status, kw)


def _call(fn, good):
    def call(**change):
        fn(**{**good, **change})

    return call


def test_attention(ops):
    good = dict(q=P, ld_q=512, k=P, ld_k=128, v=P, ld_v=128, out=P, ld_out=512, lse=P, type=1, q_start=P, k_start=P, k_len=P,
                n_seqs=2, total_q=10, kv_rows=100, max_q=5, max_k=50, heads=8, kv_heads=2, dim=64, scale=0.125, causal=1,
                workspace=P, workspace_bytes=1 << 20)
    call = _call(ops.attention_packed, good)
    for bad in (dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(q_start=0), dict(k_start=0), dict(k_len=0), dict(type=0),
                dict(type=3), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(dim=0), dict(ld_q=511), dict(ld_k=127),
                dict(ld_v=127), dict(ld_out=511), dict(n_seqs=-1), dict(total_q=-1), dict(kv_rows=-1), dict(causal=2),
                dict(max_q=-1), dict(max_k=-1)):
        refused(ARGS, call, **bad)
    for bad in (dict(q=P + 1), dict(k=P + 1), dict(v=P + 1), dict(out=P + 1), dict(lse=P + 2), dict(q_start=P + 2), dict(k_start=P + 1),
                dict(k_len=P + 2), dict(workspace=P + 8)):
        refused(ALIGN, call, **bad)
    refused(SHAPE, call, dim=264, ld_q=8 * 264, ld_k=528, ld_v=528, ld_out=8 * 264)
    refused(SHAPE, call, total_q=(1 << 30) + 1)
    refused(SHAPE, call, total_q=1 << 29)  # times 8 heads
    refused(SHAPE, call, kv_rows=(1 << 30) + 1)
    call(n_seqs=0)
    call(total_q=0)


def test_rope(ops):
    good = dict(x=P, x_type=0, ld_x=768, bias=0, positions=P, turns=P, rot_dim=64, interleaved=0, magnitude=1.0, tokens=3, heads=8,
                kv_heads=2, dim=64, q=P, ld_q=512, k=P, ld_k=128, v=P, ld_v=128, out_type=1, slots=0, n_slots=0)
    call = _call(ops.rope_qkv, good)
    for bad in (dict(x=0), dict(q=0), dict(k=0), dict(v=0), dict(positions=0), dict(turns=0), dict(x_type=3), dict(out_type=-1),
                dict(ld_x=767), dict(ld_q=511), dict(ld_k=127), dict(ld_v=127), dict(rot_dim=63), dict(rot_dim=66), dict(rot_dim=-2),
                dict(interleaved=2), dict(tokens=-1), dict(heads=0), dict(kv_heads=0), dict(dim=0), dict(slots=P, n_slots=-1)):
        refused(ARGS, call, **bad)
    for bad in (dict(x=P + 2), dict(bias=P + 2), dict(positions=P + 2), dict(turns=P + 4), dict(q=P + 1), dict(k=P + 1), dict(v=P + 1),
                dict(slots=P + 4, n_slots=1)):
        refused(ALIGN, call, **bad)
    refused(SHAPE, call, dim=514, ld_x=1 << 14, ld_q=1 << 13, ld_k=1 << 13, ld_v=1 << 13)
    call(tokens=0)


def test_norm(ops):
    good = dict(a=P, a_type=0, ld_a=64, post=1, post_gamma=P, post_beta=0, gate=0, ld_gate=0, gate_rows=0, scale=1.0, x=P, ld_x=64,
                y=P, ld_y=64, x_type=1, pre_gamma=P, pre_beta=0, h=P, ld_h=64, h_type=2, layer=0, eps=1e-6, rows=4, cols=64)
    call = _call(ops.norm_residual_rows, good)
    for bad in (dict(a=0), dict(y=0, h=0), dict(ld_a=63), dict(ld_x=63), dict(ld_y=63), dict(ld_h=63), dict(gate=P, ld_gate=63, gate_rows=1),
                dict(gate=P, ld_gate=64, gate_rows=0), dict(a_type=3), dict(x_type=-1), dict(h_type=3), dict(rows=-1), dict(cols=0),
                dict(eps=-1.0), dict(eps=math.nan), dict(post=2), dict(layer=-1)):
        refused(ARGS, call, **bad)
    for bad in (dict(a=P + 2), dict(x=P + 1), dict(y=P + 1), dict(h=P + 1), dict(post_gamma=P + 2), dict(pre_gamma=P + 1),
                dict(gate=P + 2, ld_gate=64, gate_rows=1)):
        refused(ALIGN, call, **bad)
    refused(SHAPE, call, rows=1 << 31)
    call(rows=0)


def test_8_bit(ops):
    good = dict(x=P, x_type=0, ld_x=64, codes=P, ld_codes=64, scales=P, rows=4, cols=64)
    call = _call(ops.quantize_rows_i8, good)
    for bad in (dict(x=0), dict(codes=0), dict(scales=0), dict(ld_x=63), dict(ld_codes=63), dict(x_type=5), dict(rows=-1), dict(cols=0)):
        refused(ARGS, call, **bad)
    refused(ALIGN, call, x=P + 2)
    refused(ALIGN, call, scales=P + 2)
    refused(SHAPE, call, rows=1 << 31)
    call(rows=0)
    good = dict(A=P, lda=64, scale_a=P, B=P, ldb=64, scale_b=P, bias=0, out=P, ld_out=32, out_type=1, M=4, N=32, K=64)
    call = _call(ops.i8gemm, good)
    for bad in (dict(A=0), dict(B=0), dict(scale_a=0), dict(scale_b=0), dict(out=0), dict(lda=48), dict(ldb=48), dict(ld_out=31),
                dict(out_type=3), dict(M=-1), dict(N=-1), dict(K=0)):
        refused(ARGS, call, **bad)
    for bad in (dict(A=P + 8), dict(B=P + 1), dict(lda=72), dict(ldb=72), dict(scale_a=P + 1), dict(scale_b=P + 2), dict(bias=P + 2),
                dict(out=P + 1)):
        refused(ALIGN, call, **bad)
    refused(SHAPE, call, K=131072, lda=131072, ldb=131072)
    refused(SHAPE, call, M=(1 << 30) + 1)
    refused(SHAPE, call, N=(1 << 30) + 1, ld_out=1 << 31)
    call(M=0)
    call(N=0)


def test_rope_turns(ops):
    """The plan against its formulas: plain, all pairs slower, a larger base, the ramp between both ends."""
    two_pi = 2 * math.pi
    plain, m = ops.rope_turns(128, 10000.0)
    assert m == 1.0 and len(plain) == 64
    for i, f in enumerate(plain):
        assert f == pytest.approx(10000.0 ** (-i / 64) / two_pi, rel=1e-14)
    slow, m = ops.rope_turns(128, 10000.0, ops.ROPE_LINEAR, 4.0)
    assert m == 1.0 and all(a == pytest.approx(b / 4, rel=1e-14) for a, b in zip(slow, plain))
    base, m = ops.rope_turns(128, 10000.0, ops.ROPE_BASE, 4.0)
    assert m == 1.0 and base[0] == plain[0] and base[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)
    ramp, m = ops.rope_turns(128, 10000.0, ops.ROPE_RAMP, 16.0, 4096.0)
    assert m == pytest.approx(1 + 0.1 * math.log(16.0), rel=1e-6)
    for f, p in zip(ramp, plain):
        over = p * 4096  # turns over the trained length
        if over > 40:
            assert f == p
        elif over < 0.8:
            assert f == pytest.approx(p / 16, rel=1e-14)
        else:
            assert p / 16 * (1 - 1e-14) <= f <= p
    assert sum(p / 16 * 1.0001 < f < p * 0.9999 for f, p in zip(ramp, plain)) > 10
    for bad in (dict(rot_dim=63), dict(rot_dim=0), dict(rot_dim=514), dict(rot_dim=64, base=0.0), dict(rot_dim=64, factor=0.5),
                dict(rot_dim=64, scaling=4), dict(rot_dim=64, scaling=ops.ROPE_RAMP), dict(rot_dim=64, base=math.nan),
                dict(rot_dim=64, scaling=ops.ROPE_RAMP, factor=2.0, trained_len=100.0, fast=1.0, slow=1.0)):
        refused(ARGS, ops.rope_turns, **bad)
