"""Calls of the decoder-block entry points at the limits of their index arithmetic and calls that cannot be done in place (no
GPU needed: they end at their checks)."""
import pytest

from test_decoder_refusals import ARGS, P, SHAPE, _call, ops, refused  # noqa: F401

NORM = dict(a=P, a_type=0, ld_a=64, post=1, post_gamma=P, post_beta=0, gate=0, ld_gate=0, gate_rows=0, scale=1.0, x=2 * P, ld_x=64,
            y=3 * P, ld_y=64, x_type=1, pre_gamma=P, pre_beta=0, h=4 * P, ld_h=64, h_type=2, layer=0, eps=1e-6, rows=4, cols=64)


@pytest.mark.parametrize("cols", [(1 << 30) + 1, (1 << 31) - 257, (1 << 31) - 1])
def test_rows_too_wide_for_32_bit_columns(ops, cols):  # noqa: F811
    """A block's threads step over the columns by their number: beyond 2^31 - 256 the step after the last would be negative."""
    wide = dict(ld_a=1 << 31, ld_x=1 << 31, ld_y=1 << 31, ld_h=1 << 31)
    refused(SHAPE, _call(ops.norm_residual_rows, {**NORM, **wide}), cols=cols)
    refused(SHAPE, ops.quantize_rows_i8, P, 0, 1 << 31, P, 1 << 31, P, 1, cols)


def test_query_rows_whose_blocks_pass_32_bits(ops):  # noqa: F811
    """The last block of 16 rows, and the four behind it, are numbered too: 2^31 - 65 tokens x heads is the most."""
    good = dict(q=P, ld_q=64, k=P, ld_k=8, v=P, ld_v=8, out=P, ld_out=64, lse=P, type=1, q_start=P, k_start=P, k_len=P, n_seqs=1,
                total_q=(1 << 28) - 8, kv_rows=100, max_q=1, max_k=50, heads=8, kv_heads=1, dim=8, scale=0.125, causal=1)
    call = _call(ops.attention_packed, good)
    for total_q in ((1 << 28) - 8, (1 << 28) - 1):
        refused(SHAPE, call, total_q=total_q)
    refused(SHAPE, call, total_q=(1 << 31) // 9, heads=9, ld_q=72, ld_out=72)


def test_norm_in_place_needs_the_same_layout(ops):  # noqa: F811
    """An output over an input whose elements or rows lie otherwise would overwrite what other threads still read; y and h
    over each other have no result."""
    call = _call(ops.norm_residual_rows, NORM)
    for bad in (dict(y=2 * P, ld_y=72), dict(y=2 * P, ld_x=72), dict(y=P), dict(h=P), dict(y=P, a_type=1, ld_y=72), dict(h=2 * P, ld_h=72),
                dict(h=2 * P, h_type=0), dict(h=P, h_type=0, ld_a=72), dict(h=3 * P), dict(h=3 * P, h_type=1)):
        refused(ARGS, call, **bad)
