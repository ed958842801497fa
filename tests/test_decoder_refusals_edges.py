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
