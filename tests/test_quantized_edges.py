"""Edges of the 4-bit weight path that show without a GPU: what the sources say, and what the host decides."""
import pytest
import torch

from test_wait_rules import kernels as sources


def body_of(name):
    return next(body for n, _, body in sources() if n == name)


def test_chosen_rows_are_read_after_the_wait():
    """``add_rmsnorm_q8(rows=...)`` takes indices from anywhere, the kernel launched just before it among them."""
    body = body_of("add_rmsnorm_q8_kernel")
    assert body.index("pdl_wait(pending, rows)") < body.index("rows[")
