"""How exact the fp32 gradients of the attention cores are.  They add up score gradients, or row sums of them, that cancel; the general tests hold them to
2^-15 of the sum of magnitudes.  Here the bounds are in roundings (2^-24) of a row's own magnitude m_i = sum_j p_ij (|dO| |v|^T)_ij, for inputs where an
error of the same sign in every row would show."""
import pytest
import torch

from test_attention_maps import TYPES, make, run


def _rows(q, k, v, do, scale):
    """Per (head, row): r = sum p dp and its magnitude, in 64 bits; one sample at a time."""
    t = lambda x: x.double().transpose(0, 1)
    r, m = [], []
    for i in range(q.shape[0]):
        p = torch.softmax(t(q[i]) @ t(k[i]).transpose(1, 2) * scale, -1)
        r.append((p * (t(do[i]) @ t(v[i]).transpose(1, 2))).sum(-1))
        m.append((p * (t(do[i]).abs() @ t(v[i]).abs().transpose(1, 2))).sum(-1))
    return torch.cat(r, 1), torch.cat(m, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("B, Sq, Sk", [(4, 3869, 2657), (150, 100, 107)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64])
def test_gradient_of_lam_over_many_rows(D, t, B, Sq, Sk):
    """About 15 000 rows, by two passes and as short rows.  A dp is off by about a rounding of its terms, independently from key to key and row to row; a row
    averages over 30 keys and more, so its sum is off by 1 / sqrt(30) of a rounding of m_i at most, and the rows' sum by that share of the root of the sum of
    m_i^2: under a quarter.  Sums of the matrix pipe that are cut off to one side (fp16: 2^-27 of their terms and more) would make 0.3 to 0.6 of it."""
    q, k, v, w, bk, do = make("diff", TYPES[t], B, 3, 3, D, Sq, Sk, seed=41)
    got = run("diff", q, k, v, w, bk, do)["dw"].double()
    r, m = _rows(q[:, :, :, 1], k[:, :, :, 1], v, do, D ** -0.5)
    off = (got + r.sum(1)).abs() / (2.0 ** -24 * m.square().sum(1).sqrt())
    assert float(off.max()) < 0.25, off


@pytest.mark.gpu
@pytest.mark.parametrize("B, Sq, Sk, Hkv", [(40, 16, 1500, 2), (3, 700, 900, 1), (60, 100, 107, 2)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_gradient_of_a_bucket_that_holds_whole_rows(D, t, B, Sq, Sk, Hkv):
    """One bucket for every position: a row's score gradients add up to 0, and so does the table's.  With s the sum of the row's p in fp32, S that of p dp and
    r = fl(S / s), what remains of a row is S fl(1 / s) - r s fl(1 / s): two roundings of |r| <= m_i, of the quotients, whatever their sign.  The bias of 100
    makes the row statistics 2^-18 coarse, and dp has a large mean: an r that does not fit the row's p by as much would be 20 roundings off in every row."""
    q, k, v, w, bk, do = make("relpos", TYPES[t], B, 2, Hkv, D, Sq, Sk, seed=42, buckets=4, reach=2)
    bk, w = torch.zeros_like(bk), torch.full_like(w, 100.0)
    v, do = (v.float() + 2).to(v.dtype), (do.float() * 0.1 + 1).to(do.dtype)
    got = run("relpos", q, k, v, w, bk, do)["dw"].double()
    r, m = _rows(q, k.repeat_interleave(2 // Hkv, 2), v.repeat_interleave(2 // Hkv, 2), do, D ** -0.5)
    off = got[0].abs() / (2.0 ** -24 * m.sum(1))
    assert float(off.max()) < 2 and not got[1:].any(), off
