"""A token of more query elements than the window kernel's 32-bit offsets reach
is refused, before any device call; the widest that fits is not refused for it."""

import pytest

import test_window_refusals as window
from test_int4_refusals import On


@pytest.mark.parametrize("head_dim", [64, 128])
def test_tokens_past_32_bit_offsets_are_refused(head_dim):
    from microinfer import _microinfer as m
    heads = (1 << 31) // head_dim
    big = On(1 << 40, 1 << 50)
    args = window.args(q=big, out=On(1 << 40, 1 << 52), seq_q=1, seq_k=1, kv_heads=1,
                       head_dim=head_dim)
    for over in (heads, 2 * heads - 1):
        with pytest.raises(ValueError, match="query elements a token"):
            m.device.attention_window(**{**args, "heads": over})
        with pytest.raises(ValueError, match="query elements a token"):
            m.device.attention_window_partials(1, 1, over, 1, head_dim)
    m.device.attention_window_partials(1, 1, heads - 1, 1, head_dim)
