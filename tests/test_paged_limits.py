"""Limits of the paged serving operators that need no GPU."""
from test_paged_ops import sample
from vibethinker_webgpu_lora_b200 import _lib as L


def test_the_longest_row():
    assert sample(n=(1 << 20) + 1, ld=1 << 21) == L.EG_ERR_ARG
    assert sample(rows=0, n=1 << 20, ld=1 << 20) == L.EG_OK
