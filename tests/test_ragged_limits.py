"""Sizes past what one launch of a ragged batch's operators has threads for: refused
before a launch, with no device call. A launch has fewer than 2^32 threads."""

import pytest

from test_int4_refusals import On
from test_ragged_refusals import append_args, device

FAR = 1 << 50  # bytes between buffers, more than any of them has


def test_append_refuses_more_rows_than_a_launch_takes():
    most = 0xFFFFFF * 32  # 32 rows to a workgroup of 256
    sizes = dict(heads=1, kv_heads=1, head_dim=2, k_out=None,
                 **{name: On(1 << 34, (i + 1) * FAR) for i, name in enumerate(("q", "k", "v", "q_out"))})
    for rows in (most + 1, (1 << 31) - 1):
        with pytest.raises(ValueError, match=f"at most {most} rows"):
            device().append_batch(**append_args(rows=rows, **sizes))


def test_quantise_refuses_more_rows_than_a_launch_takes():
    for features, most in ((16, 4 * 0xFFFFFF), (2048, 4 * 0xFFFFFF), (2064, 0xFFFFFF), (65536, 0xFFFFFF)):
        x, codes = On(1 << 46, FAR), On(1 << 46, 2 * FAR, 1)
        with pytest.raises(ValueError, match=f"at most {most} rows of {features} values"):
            device().quantise_rows_int8(x, codes, On(1 << 30, 3 * FAR, 4), most + 1, features)


@pytest.mark.parametrize("hd,kv,most", [(64, 128, (1 << 23) - 1), (128, 256, (1 << 24) - 1)])
def test_packed_attention_refuses_more_tiles_than_a_launch_takes(hd, kv, most):
    """65,535 sequences of a token: a tile each of every KV head, and a 128th more."""
    rows = 65535
    far = lambda i: On(1 << 40, i * FAR)  # noqa: E731
    with pytest.raises(ValueError, match=f"at most {most} tiles"):
        device().attention_packed(far(1), far(2), far(3), far(4), On(rows + 1, 5 * FAR, 4), None, rows, rows,
                                  rows, kv, kv, hd)
