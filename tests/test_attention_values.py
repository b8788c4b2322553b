"""Values that the attention cores meet at the edges: rows of a cache that no query sees.  The formulas in 64 bits and their tolerances are those of
test_attention_maps."""
import math

import pytest
import torch

from test_attention_maps import OPS, check, make, mask, reference, run


def _spoil(x, at, value):
    x = x.clone()
    x[at] = value
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("Sq, Sk, seen", [(1, 300, 130), (1, 90, 1), (5, 2000, 777), (33, 700, 333), (70, 100, 81), (100, 128, 100), (150, 400, 201), (150, 260, 192), (9, 70, 0)])
@pytest.mark.parametrize("op, D", OPS)
def test_keys_that_no_query_sees_may_hold_anything(op, D, Sq, Sk, seen):
    """A cache with room behind the newest token, whose rows there were never written: the causal mask hides them from every query."""
    for Hkv in (2, 4):
        q, k, v, w, bk, do = make(op, torch.bfloat16, 2, 4, Hkv, D, Sq, Sk, seed=32, buckets=8, reach=40)
        for kvalid in (None, mask("holes", 2, Sk)):
            opts = dict(kvalid=kvalid, causal=True, q_offset=seen - Sq)
            want = run(op, q, k, v, w, bk, do, **opts)
            check(want, reference(op, q, k, v, w, bk, do=do, **opts))
            for x in (math.nan, math.inf):
                k2, v2 = _spoil(k, (slice(None), slice(seen, None)), x), _spoil(v, (slice(None), slice(seen, None)), x)
                got = run(op, q, k2, v2, w, bk, do, **opts)
                assert all(torch.equal(got[n], want[n]) for n in got), x
                assert not got["dk"][:, seen:].any() and not got["dv"][:, seen:].any()
