"""Values that the attention cores meet at the edges: NaN and infinities that are not masked, rows of a cache that no query sees, small gradients, the
largest tables.  The formulas in 64 bits and their tolerances are those of
test_attention_maps."""
import math

import pytest
import torch

from test_attention_maps import OPS, TYPES, both, check, make, mask, reference, run


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


@pytest.mark.gpu
@pytest.mark.parametrize("Sq, Sk, H, Hkv", [(70, 100, 2, 2), (70, 100, 4, 2), (150, 201, 2, 2), (5, 700, 4, 2)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("op, D", OPS)
def test_nan_and_infinity_reach_what_depends_on_them(op, D, what, t, Sq, Sk, H, Hkv):
    """One in a query, an unmasked key, a value or an output gradient: none of what the formula makes of it comes out finite, in either backward form; masked
    keys' gradients are zeros, and what does not depend on it keeps its bits."""
    q, k, v, w, bk, do = make(op, TYPES[t], 2, H, Hkv, D, Sq, Sk, seed=31, buckets=8, reach=40)
    kv = mask("holes", 2, Sk)
    kv[:, 3] = 1
    b, h, i, j, R = 1, 1, Sq // 2, 3, 40
    kh = h * Hkv // H
    valid = kv[b] != 0
    heads = [h] if what in ("q", "do") else [x for x in range(H) if x * Hkv // H == kh]
    want = run(op, q, k, v, w, bk, do, kvalid=kv)
    for value in (math.nan, math.inf):
        for m in (0, 1) if op == "diff" and what in ("q", "k") else (0,):
            x = dict(q=q, k=k, v=v, do=do)
            at = (b, i, h) if what in ("q", "do") else (b, j, kh)
            x[what] = _spoil(x[what], at + ((m, 5) if x[what].dim() == 5 else (5,)), value)
            got = run(op, x["q"], x["k"], x["v"], w, bk, x["do"], kvalid=kv)
            bad = {n: ~y.isfinite() for n, y in got.items()}
            rows = torch.ones(Sq, dtype=torch.bool, device="cuda") if what in ("k", "v") else torch.arange(Sq, device="cuda") == i
            for hd in heads:
                lost = rows                                  # rows without a finite score map: a key of +inf takes all of a row, one of -inf leaves it
                if what == "k" and value == math.inf:
                    lost = rows & ((q[b, :, hd, m, 5] if op == "diff" else q[b, :, hd, 5]) > 0)
                assert bool(bad["dq"][b, :, hd].flatten(1).any(1)[lost].all()) and not bool(bad["dq"][b, :, hd][~rows].any())
                if what != "do":
                    assert bool(bad["o"][b, :, hd].any(1)[lost].all()) and not bool(bad["o"][b, :, hd][~rows].any())
                if what in ("q", "k"):
                    assert bool((got["lse"][b, hd, m] if op == "diff" else got["lse"][b, hd]).isnan()[lost].all())
                if op == "relpos":
                    rel = (torch.arange(Sk, device="cuda")[valid][None] - torch.arange(Sq, device="cuda")[lost][:, None]).clamp(-R, R) + R
                    assert bool(bad["dw"][bk.long()[rel].unique(), hd].all())
                elif m == 1 or what in ("v", "do"):          # (lam's gradient is the second map's)
                    assert bool(bad["dw"][hd])
            dk = bad["dk"][b, :, kh, m] if op == "diff" else bad["dk"][b, :, kh]
            assert bool(dk.any(1)[valid].all())
            if what == "v":
                assert torch.equal(got["dv"], want["dv"])
            else:
                assert bool(bad["dv"][b, :, kh].any(1)[valid].all())
            assert not got["dk"][b][~valid].any() and not got["dv"][b][~valid].any()
            rest, rest_k = [y for y in range(H) if y not in heads], [y for y in range(Hkv) if y != kh]
            for n, other in (("o", rest), ("dq", rest), ("dk", rest_k), ("dv", rest_k)):
                assert torch.equal(got[n][0], want[n][0]) and torch.equal(got[n][:, :, other], want[n][:, :, other]), n


@pytest.mark.gpu
@pytest.mark.parametrize("Sq, Sk, H, Hkv", [(100, 100, 2, 2), (60, 128, 4, 2), (1000, 1000, 2, 1), (700, 4000, 2, 2)])
@pytest.mark.parametrize("power", [-6, -10, -13])
@pytest.mark.parametrize("op, D", OPS)
def test_small_gradients_in_half_precision(op, D, power, Sq, Sk, H, Hkv):
    """Output gradients of 2^power, as a mean over a batch leaves them without a loss scale: dq and dk are about as near to the formula as at 2^0, where the
    score gradients lie in the type's normal range.  In the 2-norm an error of P, dS or the output itself is at most u sqrt(1 / 3) of its part, three of
    them 2^-11, and a rounding of the output below the normal range adds 2^-25 sqrt(1 / 3) per entry; twice their sum is allowed."""
    q, k, v, w, bk, do = make(op, torch.float16, 1, H, Hkv, D, Sq, Sk, seed=33)
    rows = torch.rand(1, Sq, 1, 1, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.9
    do = torch.where(rows, do, do * 2.0 ** -4) * 2.0 ** power                        # (some rows smaller still)
    got, want = run(op, q, k, v, w, bk, do), reference(op, q, k, v, w, bk, do=do)
    for n in ("dq", "dk"):
        x = want[n][0]
        bound = 2 * (2.0 ** -11 * x.norm() + 2.0 ** -25 * (x.numel() / 3) ** 0.5)
        assert (got[n].double() - x).norm() < bound, (n, float((got[n].double() - x).norm() / bound))
    check({n: got[n] for n in ("o", "lse", "dv", "dw")}, want)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq, Sk", [(90, 110), (200, 300)])
@pytest.mark.parametrize("op, D", OPS)
def test_powers_of_two_pass_through(op, D, Sq, Sk):
    """Gradients are linear in dO: halving it halves the fp32 gradients exactly, and those in 16 bits as long as no entry leaves the normal range."""
    q, k, v, w, bk, do = make(op, torch.float16, 2, 2, 2, D, Sq, Sk, seed=34)
    do = (do.clamp(-3, 3) * 256).round() / 1024              # (whole multiples of 2^-10, at most 3 / 4: their halves are exact)
    one, half = run(op, q, k, v, w, bk, do), run(op, q, k, v, w, bk, do * 0.5)
    assert torch.equal(one["dw"], half["dw"] * 2)
    for n in ("dq", "dk", "dv"):
        big = one[n].abs() >= 2.0 ** -13
        assert torch.equal(one[n][big], half[n][big] * 2), n


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 128])
def test_largest_reach_and_table(D):
    """The largest window that a workgroup holds, and the most positions and buckets that the table's gradient adds up, one position per bucket."""
    q, k, v, _, _, do = make("relpos", torch.bfloat16, 1, 1, 1, D, 4300, 4200, seed=35)
    w = torch.randn(8192, 1, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    bk = torch.arange(2 * 4095 + 1, dtype=torch.int32, device="cuda")
    both("relpos", q, k, v, w, bk, do, q_offset=-50)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq, Sk", [(1, 900), (20, 3000), (70, 100), (140, 160)])
@pytest.mark.parametrize("op, D", OPS)
def test_repeats_and_gradients_that_are_not_asked_for(op, D, Sq, Sk):
    """Split keys, short rows, two passes: the same bits every time, with and without the gradient of the table or of lam."""
    from univtg_amd import ops
    q, k, v, w, bk, do = make(op, torch.float16, 3, 4, 4, D, Sq, Sk, seed=36)
    opts = dict(kvalid=mask("prefix", 3, Sk), causal=True, q_offset=Sk - Sq)
    a = run(op, q, k, v, w, bk, do, **opts)
    for _ in range(3):
        b = run(op, q, k, v, w, bk, do, **opts)
        assert all(torch.equal(a[n], b[n]) for n in a)
    if op == "relpos":
        got = ops.relpos_attention_bwd(do, q, k, v, w, bk, a["o"], a["lse"], need_dtable=False, **opts)
    else:
        o2 = ops.diff_attention_fwd(q, k, v, w, need_o2=True, **opts)[2]
        got = ops.diff_attention_bwd(do, q, k, v, w, a["o"], o2, a["lse"], need_dlam=False, **opts)
    assert got[3] is None and all(torch.equal(x, a[n]) for x, n in zip(got, ("dq", "dk", "dv")))
