"""Sizes at the ends of the token-path entry points' index ranges, refused before
anything is launched (no GPU)."""
from __future__ import annotations


from test_token_ops_host import EUNSUPPORTED, FLT, I64, INT, PTR, lib  # noqa: F401


def test_rotary_refuses_heads_whose_index_would_wrap(lib):  # noqa: F811
    """A block's threads count a token's elements in steps of 256 in 32 bits: 42966
    heads of 49981 elements (2^31 - 2) would step past the end."""
    p = PTR(256)

    def call(heads, dim):
        return lib.pkv_rotary(p, I64(heads * dim), I64(dim), INT(heads), p, I64(heads * dim),
                              I64(dim), p, I64(dim), I64(dim), INT(0), p, I64(dim), I64(dim),
                              INT(0), I64(1), INT(dim), p, INT(1), p, None, INT(0), INT(0),
                              FLT(1.0), INT(0), None)
    assert call(42966, 49981) == EUNSUPPORTED
    assert call(65536, 32768) == EUNSUPPORTED        # 2^31
