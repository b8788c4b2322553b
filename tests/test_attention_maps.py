"""Attention with a learned relative position bias by buckets, and differential attention: kernels against the formulas in 64 bits.

Tolerances are derived, elementwise.  u = eps / 2 of the operands' type is the relative error of one rounding, t = 2^-25 (fp16) the absolute one of
a rounding that leaves the normal range.  The kernels round the probabilities once for the product with v (and with dO), the score gradients once
for the products with k and q, and every output once; scores, exponentials and sums are fp32, whose errors (products of up to 128 terms, an exponent
of a size up to about 2^5, sums of some thousand terms in a tree of MFMA and lane sums) stay under c = 2^-15 of the sum of magnitudes.  So
    |o - o*|   <= (u + c) P|v| + t sum|v| + u |o*|                         P|v|: the product with magnitudes
    |dv - dv*| <= (u + c) P^T|dO| + t sum|dO| + u |dv*|
    |dk - dk*| <= scale ((u + c) M^T|q| + t sum|q|) + u |dk*|               M = P (|dO||v|^T + |r|), at least |dS|
    |dq - dq*| <= scale ((u + c) M + P e)|k| + ... + u |dq*|                 e = |dO| (bound of o): that pass takes r from the rounded o
and the fp32 outputs stay within c of their sums of magnitudes."""
import ctypes as C
import math

import pytest
import torch

C_ACC = 2.0 ** -15
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- the formulas in 64 bits ------------------------------------------------------------------------------------------------------------
def _hide(B, Sq, Sk, kvalid, causal, off, dev):
    h = torch.zeros(B, 1, Sq, Sk, dtype=torch.bool, device=dev)
    if causal:
        h |= (torch.arange(Sk, device=dev)[None] > torch.arange(Sq, device=dev)[:, None] + off)[None, None]
    if kvalid is not None:
        h |= (kvalid == 0)[:, None, None]
    return h


def _heads(x, H):
    return x.double().transpose(1, 2).repeat_interleave(H // x.shape[2], 1)


def _softmax(x, hide):
    x = x.masked_fill(hide, -math.inf)
    m = x.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
    p = torch.exp(x - m)
    s = p.sum(-1, keepdim=True)
    return p / s.clamp_min(1e-300), (torch.log(s) + m)[..., 0]


def _clean(x, kvalid):
    """x with the rows of masked keys zeroed: they may hold anything and must not matter."""
    return x if kvalid is None else torch.where((kvalid != 0).view(*kvalid.shape, *([1] * (x.dim() - 2))), x, torch.zeros_like(x))


def reference(op, q, k, v, w, buckets=None, kvalid=None, q_offset=0, causal=False, scale=None, do=None):
    """Outputs and gradients in 64 bits, each with the elementwise tolerance of the module's comment: {name: (value, tolerance)}."""
    B, Sq, H = q.shape[:3]
    Sk, Hkv, D, t = k.shape[1], k.shape[2], q.shape[-1], q.dtype
    u, tiny = torch.finfo(t).eps / 2, (2.0 ** -25 if t == torch.float16 else 0.0)
    G, dev, scale = H // Hkv, q.device, D ** -0.5 if scale is None else scale
    hide = _hide(B, Sq, Sk, kvalid, causal, q_offset, dev)
    k, v = _clean(k, kvalid), _clean(v, kvalid)
    V, w = _heads(v, H), w.double()
    if op == "relpos":
        R = buckets.numel() // 2
        rel = (torch.arange(Sk, device=dev)[None] - torch.arange(Sq, device=dev)[:, None] - q_offset).clamp(-R, R) + R
        idx = buckets.long()[rel]
        Q, K = [_heads(q, H)], [_heads(k, H)]
        x = [Q[0] @ K[0].transpose(2, 3) * scale + w[idx].permute(2, 0, 1)[None]]
        coef = [torch.ones(1, H, 1, 1, dtype=torch.float64, device=dev)]
    else:
        Q, K = [_heads(q[:, :, :, m], H) for m in (0, 1)], [_heads(k[:, :, :, m], H) for m in (0, 1)]
        x = [a @ b.transpose(2, 3) * scale for a, b in zip(Q, K)]
        coef = [torch.ones(1, H, 1, 1, dtype=torch.float64, device=dev), -w.view(1, H, 1, 1)]
    P, lse = zip(*[_softmax(s, hide) for s in x])
    O = [p @ V for p in P]
    back = lambda z: z.transpose(1, 2)
    o = sum(c * y for c, y in zip(coef, O))
    tol_m = [(u + C_ACC) * (p @ V.abs()) + tiny * V.abs().sum(2, keepdim=True) for p in P]
    tol_o = sum(c.abs() * y for c, y in zip(coef, tol_m)) + u * o.abs() + tiny
    big = scale * sum(a.abs() @ b.abs().transpose(2, 3) for a, b in zip(Q, K)).amax().item()
    LSE = lse[0] if op == "relpos" else torch.stack(lse, 2)
    out = {"o": (back(o), back(tol_o)), "lse": (LSE, 2.0 ** -20 * (4 + big + LSE.abs().nan_to_num(posinf=0.0)))}
    if do is None:
        return out
    g = do.double().transpose(1, 2)
    dp, mag = g @ V.transpose(2, 3), g.abs() @ V.abs().transpose(2, 3)
    Pd = sum(c * p for c, p in zip(coef, P))
    share = lambda z: z.view(B, Hkv, G, *z.shape[2:]).sum(2).transpose(1, 2)
    dv = share(Pd.transpose(2, 3) @ g)
    Pabs = sum(c.abs() * p for c, p in zip(coef, P))
    tol = share(((u + C_ACC) * Pabs.transpose(2, 3)) @ g.abs() + tiny * g.abs().sum(2, keepdim=True))
    out["dv"] = (dv, tol + u * dv.abs() + tiny)
    dq, dk, tq, tk, ds_, mag_ = [], [], [], [], [], []
    # the pass over queries takes the row sums from the rounded outputs (of both maps)
    e = [(g.abs() * (sum(tol_m[j] * coef[j].abs() for j in range(len(P))) + u * o.abs() + (tol_m[-1] + u * O[-1].abs()) * coef[-1].abs() * (len(P) - 1))).sum(-1, keepdim=True)]
    if op == "diff":
        e.append((g.abs() * (tol_m[1] + u * O[1].abs())).sum(-1, keepdim=True))
    for m in range(len(P)):
        r = (P[m] * dp).sum(-1, keepdim=True)
        ds = coef[m] * P[m] * (dp - r)
        M = coef[m].abs() * P[m] * (mag + (P[m] * mag).sum(-1, keepdim=True))
        dq.append(back(scale * (ds @ K[m])))
        tq.append(back(scale * (((u + C_ACC) * M + coef[m].abs() * P[m] * e[m]) @ K[m].abs() + tiny * K[m].abs().sum(2, keepdim=True))))
        dk.append(share(scale * (ds.transpose(2, 3) @ Q[m])))
        tk.append(share(scale * (((u + C_ACC) * M).transpose(2, 3) @ Q[m].abs() + tiny * Q[m].abs().sum(2, keepdim=True))))
        ds_.append(ds)
        mag_.append(M)
    join = (lambda z: z[0]) if op == "relpos" else (lambda z: torch.stack(z, 3))
    for n, val, tol in (("dq", join(dq), join(tq)), ("dk", join(dk), join(tk))):
        out[n] = (val, tol + u * val.abs() + tiny)
    if op == "relpos":
        flat = idx.reshape(-1)
        sums = [torch.zeros(w.shape[0], H, dtype=torch.float64, device=dev).index_add_(0, flat, z.sum(0).permute(1, 2, 0).reshape(-1, H)) for z in (ds_[0], mag_[0])]
        out["dw"] = (sums[0], C_ACC * sums[1] + 1e-30)
    else:
        r2 = (P[1] * dp).sum((0, 2, 3))
        out["dw"] = (-r2, C_ACC * (P[1] * mag).sum((0, 2, 3)) + 1e-30)
    return out


def check(got, want):
    for n, x in got.items():
        val, tol = want[n]
        assert x.shape == val.shape, (n, x.shape, val.shape)
        x = x.double()
        same = x == val                                     # infinities
        bad = ~(same | ((x - val).abs() <= tol))
        if bad.any():
            at = torch.nonzero(bad)[0].tolist()
            raise AssertionError(f"{n}: {int(bad.sum())} of {x.numel()} off, first at {at}: {float(x[tuple(at)])} for {float(val[tuple(at)])}, tolerance {float(tol[tuple(at)])}")


# ---- inputs -----------------------------------------------------------------------------------------------------------------------------
def make(op, t, B, H, Hkv, D, Sq, Sk, seed=0, buckets=32, reach=128, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)
    m = (2,) if op == "diff" else ()
    q, k, v = n(B, Sq, H, *m, D).to(t), n(B, Sk, Hkv, *m, D).to(t), n(B, Sk, Hkv, D * (2 if m else 1)).to(t)
    do = n(B, Sq, H, v.shape[-1]).to(t)
    if op == "relpos":
        from univtg_amd import ops
        return q, k, v, n(buckets, H), ops.relpos_buckets(buckets, reach, device=dev), do
    return q, k, v, torch.rand(H, generator=g, device=dev) + 0.1, None, do


def run(op, q, k, v, w, buckets, do, **opts):
    from univtg_amd import ops
    if op == "relpos":
        o, lse = ops.relpos_attention_fwd(q, k, v, w, buckets, **opts)
        dq, dk, dv, dw = ops.relpos_attention_bwd(do, q, k, v, w, buckets, o, lse, **opts)
    else:
        o, lse, o2 = ops.diff_attention_fwd(q, k, v, w, need_o2=True, **opts)
        dq, dk, dv, dw = ops.diff_attention_bwd(do, q, k, v, w, o, o2, lse, **opts)
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv, "dw": dw}


def both(op, q, k, v, w, buckets, do, **opts):
    check(run(op, q, k, v, w, buckets, do, **opts), reference(op, q, k, v, w, buckets, do=do, **opts))


def mask(kind, B, Sk, seed=1):
    if kind == "none":
        return None
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "holes":
        return (torch.rand(B, Sk, generator=g, device="cuda") < 0.6).to(torch.uint8)
    if kind == "first":                                      # one key, the last one
        m = torch.zeros(B, Sk, dtype=torch.uint8, device="cuda")
        m[:, -1] = 1
        return m
    lens = torch.randint(1, Sk + 1, (B,), generator=g, device="cuda")
    if kind == "empty":                                      # a padded batch whose first sample has no key at all
        lens[0] = 0
    return (torch.arange(Sk, device="cuda")[None] < lens[:, None]).to(torch.uint8)


HEADS = {"relpos": (32, 64, 128), "diff": (32, 64)}
OPS = [(op, D) for op in HEADS for D in HEADS[op]]


# ---- CPU: the host side -------------------------------------------------------------------------------------------------------------------
def test_relpos_buckets_borders():
    from univtg_amd import ops
    for n, reach, both_ways in ((32, 128, True), (32, 128, False), (16, 64, True), (48, 400, True), (4, 3, True), (3, 2, False), (64, 1024, False)):
        b = ops.relpos_buckets(n, reach, both_ways, device="cpu").tolist()
        assert len(b) == 2 * reach + 1 and min(b) >= 0 and max(b) < n
        half = n // 2 if both_ways else n
        exact = half // 2
        behind = [b[reach - d] for d in range(reach + 1)]
        assert behind[:exact] == list(range(exact)) and behind[-1] == half - 1 and behind == sorted(behind)
        for d in range(exact, reach + 1):                    # the border condition itself, in whole numbers
            i = behind[d] - exact
            m = half - exact
            assert d ** m * exact ** i >= reach ** i * exact ** m
            assert i == m - 1 or d ** m * exact ** (i + 1) < reach ** (i + 1) * exact ** m
        assert b[reach + 1:] == ([half + x for x in behind[1:]] if both_ways else [0] * reach)
    for bad in ((2, 8, True), (7, 8, True), (32, 8, True), (1, 8, False)):
        with pytest.raises(ValueError):
            ops.relpos_buckets(*bad, device="cpu")


def _dims(**kw):
    from univtg_amd import _lib
    d = dict(dtype=0, B=2, H=4, Hkv=2, D=64, Sq=5, Sk=9, causal=0, q_offset=0, scale=0.1, n_buckets=32, reach=128, q_sb=0, q_ss=256, q_sh=64, k_ss=128, k_sh=64,
             v_ss=128, v_sh=64)
    return _lib.AttnDims(**dict(d, **kw))


@pytest.mark.parametrize("maps, bad, code", [
    (1, dict(B=0), -11), (1, dict(Sk=0), -11), (2, dict(Sq=-1), -11), (1, dict(dtype=2), -30), (2, dict(Hkv=3), -31), (1, dict(D=48), -5), (2, dict(D=128), -32),
    (1, dict(scale=0.0), -33), (2, dict(scale=float("inf")), -33), (1, dict(scale=float("nan")), -33), (1, dict(q_offset=1 << 30), -34), (1, dict(Sk=1 << 25), -34),
    (1, dict(q_ss=257), -35), (2, dict(k_sm=4), -35), (1, dict(v_sh=-64), -35), (1, dict(reach=0), -36), (1, dict(reach=4096), -36), (1, dict(n_buckets=0), -37),
    (1, dict(n_buckets=8193), -37), (2, dict(q_ss=(1 << 26) + 8), -38), (1, dict(k_ss=1 << 27), -38), (2, dict(v_ss=1 << 40), -38), (1, dict(kvalid_sb=-1), -35),
    (1, dict(H=65536, Hkv=1), -34), (2, dict(Sq=1 << 24, H=64, Hkv=64), -34), (1, dict(Sk=1 << 24, H=64, Hkv=64), -34),
    (1, dict(B=1 << 16, H=1 << 10, Hkv=1 << 10), -34), (1, {}, -20), (2, {}, -20)])
def test_c_abi_refuses(maps, bad, code):
    """Every refusal comes back before anything is enqueued (no GPU here, null pointers)."""
    from univtg_amd import _lib
    lib = _lib.load()
    d = C.byref(_dims(**bad))
    fwd, bwd = (lib.uvtg_relpos_attention_fwd, lib.uvtg_relpos_attention_bwd) if maps == 1 else (lib.uvtg_diff_attention_fwd, lib.uvtg_diff_attention_bwd)
    assert fwd(d, *[None] * 10) == code and bwd(d, *[None] * 15) == code
    assert lib.uvtg_strerror(code) not in (b"invalid argument", b"ok")
    for backward in (0, 1):
        assert (lib.uvtg_attn_ws_bytes(d, maps, backward) == 0) == (code != -20 or backward == 0)


def test_c_abi_refuses_misaligned_and_foreign_structs():
    from univtg_amd import _lib
    lib = _lib.load()
    d = _dims()
    p = [C.c_void_p(4096)] * 10
    for i in (0, 1, 2):                                      # q, k, v off by 8 bytes: refused, nothing is read
        a = list(p)
        a[i] = C.c_void_p(4104)
        assert lib.uvtg_relpos_attention_fwd(C.byref(d), *a) == -35
    d.struct_size -= 4
    assert lib.uvtg_relpos_attention_fwd(C.byref(d), *p) == -18 and lib.uvtg_attn_ws_bytes(C.byref(d), 1, 1) == 0
    assert lib.uvtg_diff_attention_fwd(None, *p) == -10
    assert lib.uvtg_attn_ws_bytes(C.byref(_dims()), 3, 0) == 0


def test_no_cpu_fallback():
    from univtg_amd import attention, ops
    q = torch.zeros(1, 4, 2, 32, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.relpos_attention_fwd(q, q, q, torch.zeros(4, 2), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm device"):
        attention.diff_attention(q[:, :, :, None].expand(1, 4, 2, 2, 32), q[:, :, :, None].expand(1, 4, 2, 2, 32), torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(2))


def test_capture_is_refused_while_a_foreign_graph_of_a_leaf_lives():
    from univtg_amd import attention

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, y):
            return x * 2 + y

        @staticmethod
        def backward(ctx, g):
            return g * 2, g

    x, y = torch.zeros(3, requires_grad=True), torch.zeros(3)
    alive = attention._apply(Twice, (x, y), x, y)            # noted on x for stream 0
    attention._check_capture([x], 0)
    with pytest.raises(RuntimeError, match="still holds a leaf"):
        attention._check_capture([x], 2)
    kept = alive * 3                                         # the graph lives on behind a result
    for _ in range(3):
        attention._apply(Twice, (x, y), x, y)
    assert len(x._attention_graphs) == 2                     # the graphs that died are forgotten
    del alive
    with pytest.raises(RuntimeError, match="still holds a leaf"):
        attention._check_capture([x], 2)
    del kept
    attention._check_capture([x], 2)
    assert not hasattr(y, "_attention_graphs")


def test_leaves_are_copied_and_saved_as_before():
    """What a call notes on its leaves goes through copies and files."""
    import copy
    import io

    from univtg_amd import attention

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 2

        @staticmethod
        def backward(ctx, g):
            return g * 2

    x = torch.nn.Parameter(torch.arange(3.0))
    alive = attention._apply(Twice, (x,), x)
    with io.BytesIO() as f:
        torch.save(x, f)
        f.seek(0)
        y = torch.load(f, weights_only=True)
    assert torch.equal(x, y) and torch.equal(x, copy.deepcopy(x)) and y.requires_grad
    del alive
    attention._check_capture([x, y], 5)


def test_reference_against_differences():
    """The formulas that the kernels are held to: directional derivatives of the 64-bit forward by central differences."""
    for op in ("relpos", "diff"):
        q, k, v, w, bk, do = [x.double() if torch.is_tensor(x) and x.is_floating_point() else x
                              for x in make(op, torch.float32, 2, 4, 2, 8, 5, 7, buckets=6, reach=4, dev="cpu")]
        kv = torch.tensor([[1] * 7, [1, 0, 1, 1, 0, 1, 0]])
        opts = dict(kvalid=kv, causal=True, q_offset=1)
        want = reference(op, q, k, v, w, bk, do=do, **opts)
        for n, x in (("dq", q), ("dk", k), ("dv", v), ("dw", w)):
            z = torch.randn(x.shape, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
            args = dict(q=q, k=k, v=v, w=w)
            key = n[1]
            f = [(reference(op, args["q"] if key != "q" else q + e * z, args["k"] if key != "k" else k + e * z, args["v"] if key != "v" else v + e * z,
                            args["w"] if key != "w" else w + e * z, bk, **opts)["o"][0] * do).sum() for e in (1e-5, -1e-5)]
            assert abs((f[0] - f[1]) / 2e-5 - (want[n][0] * z).sum()) < 1e-7, (op, n)


# ---- GPU ----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("op, D", OPS)
def test_lengths(op, D, t):
    """From one position to a few tiles, around the edges of 32, 64 and 128."""
    for Sq, Sk in ((1, 1), (1, 2), (2, 1), (7, 31), (32, 32), (33, 65), (63, 64), (64, 63), (127, 129), (130, 97), (200, 257)):
        both(op, *make(op, TYPES[t], 2, 2, 2, D, Sq, Sk, seed=Sq))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "prefix", "holes", "empty", "first"])
@pytest.mark.parametrize("op, D", OPS)
def test_masks(op, D, kind):
    x = make(op, torch.bfloat16, 3, 2, 2, D, 150, 201, seed=5)
    both(op, *x, kvalid=mask(kind, 3, 201))
    both(op, *x, kvalid=mask(kind, 3, 201), causal=True, q_offset=51)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [-70, -1, 0, 1, 40, 300])
@pytest.mark.parametrize("op, D", OPS)
def test_causal_offsets(op, D, off):
    """Queries ahead of, at and behind the keys: with a negative offset the first rows see nothing."""
    both(op, *make(op, torch.float16, 2, 2, 2, D, 140, 170, seed=6, reach=33), causal=True, q_offset=off)
    both(op, *make(op, torch.bfloat16, 1, 2, 2, D, 140, 170, seed=7, reach=33), q_offset=off)


@pytest.mark.gpu
@pytest.mark.parametrize("H, Hkv", [(4, 1), (6, 2), (8, 8), (12, 3)])
@pytest.mark.parametrize("op, D", OPS)
def test_shared_heads(op, D, H, Hkv):
    both(op, *make(op, torch.bfloat16, 2, H, Hkv, D, 100, 130, seed=8), kvalid=mask("prefix", 2, 130))
    both(op, *make(op, torch.float16, 2, H, Hkv, D, 3, 300, seed=9), causal=True, q_offset=297)


@pytest.mark.gpu
@pytest.mark.parametrize("buckets, reach", [(4, 2), (16, 20), (32, 128), (64, 700), (32, 3000)])
@pytest.mark.parametrize("D", HEADS["relpos"])
def test_reach(D, buckets, reach):
    """Windows inside a tile, over several tiles and beyond the sequence."""
    both("relpos", *make("relpos", torch.bfloat16, 2, 2, 2, D, 260, 333, seed=10, buckets=buckets, reach=reach), kvalid=mask("prefix", 2, 333))
    both("relpos", *make("relpos", torch.bfloat16, 1, 2, 1, D, 2, 1500, seed=11, buckets=buckets, reach=reach), q_offset=1400)


@pytest.mark.gpu
def test_any_bucket_map_and_entries_out_of_range():
    """The map is data: any assignment, and an entry outside the table reads (and adds to) the nearest row inside."""
    q, k, v, w, _, do = make("relpos", torch.bfloat16, 2, 2, 2, 64, 90, 120, seed=12, buckets=10)
    bk = torch.randint(0, 10, (2 * 17 + 1,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.int32)
    both("relpos", q, k, v, w, bk, do)
    wild = bk.clone()
    wild[3], wild[30] = -7, 1000
    tame = wild.clamp(0, 9)
    a, b = run("relpos", q, k, v, w, wild, do), run("relpos", q, k, v, w, tame, do)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.gpu
@pytest.mark.parametrize("op, D", OPS)
@pytest.mark.parametrize("B, H, Hkv, Sq, Sk", [(1, 2, 2, 1, 4000), (3, 4, 1, 1, 1000), (1, 8, 2, 5, 2500), (2, 2, 1, 33, 700), (1, 1, 1, 200, 3000), (40, 8, 8, 1, 70)])
def test_few_rows_over_long_keys(op, D, B, H, Hkv, Sq, Sk):
    x = make(op, torch.bfloat16, B, H, Hkv, D, Sq, Sk, seed=13)
    both(op, *x, kvalid=mask("empty", B, Sk), causal=True, q_offset=Sk - Sq)
    both(op, *x, kvalid=mask("holes", B, Sk))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "empty"])
@pytest.mark.parametrize("op, D", OPS)
def test_many_short_heads(op, D, kind):
    """More heads of short rows than workgroups that stay on the chip: each takes several, of other samples."""
    both(op, *make(op, torch.bfloat16, 75, 15, 15, D, 37, 70, seed=24), kvalid=mask(kind, 75, 70))


@pytest.mark.gpu
@pytest.mark.parametrize("op, D", OPS)
def test_long_rows(op, D):
    """More key tiles than a workgroup holds masks for at a time (16384 keys), and training rows of a few thousand positions."""
    q, k, v, w, bk, do = make(op, torch.bfloat16, 1, 1, 1, D, 130, 17000, seed=14)
    both(op, q, k, v, w, bk, do, kvalid=mask("holes", 1, 17000))
    both(op, *make(op, torch.bfloat16, 1, 2, 1, D, 2100, 1900, seed=15), causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_masked_rows_may_hold_anything(op):
    """Infinities, NaN and the types' largest values in masked keys' rows reach no output; gradients of those rows are zeros."""
    for Sq in (1, 70):
        q, k, v, w, bk, do = make(op, torch.bfloat16, 2, 2, 1, 64, Sq, 150, seed=16)
        m = mask("holes", 2, 150)
        want = reference(op, q, k, v, w, bk, kvalid=m, do=do)
        for i, x in enumerate((math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).max)):
            k2, v2 = k.clone(), v.clone()
            k2[m == 0], v2[m == 0] = x, x
            got = run(op, q, k2, v2, w, bk, do, kvalid=m)
            check(got, want)
            assert not got["dk"][m == 0].any() and not got["dv"][m == 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_large_and_equal_scores(op):
    """Scores of some hundreds (one key takes everything), a rising maximum along the keys, and rows of equal scores."""
    q, k, v, w, bk, do = make(op, torch.bfloat16, 1, 2, 2, 64, 70, 400, seed=17)
    ramp = torch.linspace(0.02, 3.0, 400, device="cuda").view(1, 400, 1, *([1] * (k.dim() - 3)))
    both(op, (q.abs() * 2).contiguous(), (k.abs() * ramp).to(torch.bfloat16), v, w, bk, do)
    both(op, torch.zeros_like(q), k, v, w, bk, do)


@pytest.mark.gpu
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("H, Hkv, Sq, Sk", [(2, 2, 70, 100), (4, 2, 150, 200), (2, 1, 1, 700)])
@pytest.mark.parametrize("D", HEADS["relpos"])
def test_positions_the_table_takes_out(D, H, Hkv, Sq, Sk, low):
    """Table entries of -inf, and of the type's lowest value: some positions, all of one head's, and the outermost buckets of another."""
    q, k, v, w, bk, do = make("relpos", torch.bfloat16, 2, H, Hkv, D, Sq, Sk, buckets=8, reach=40)
    kv = mask("holes", 2, Sk)
    off = Sk - Sq
    gone = torch.zeros(w.shape, dtype=torch.bool, device="cuda")
    gone[1::3, 0] = True                                     # (buckets behind the query and ahead of it)
    gone[:, 1] = True
    if H > 2:
        gone[bk[0].item(), 2] = gone[bk[-1].item(), 2] = True
    got = run("relpos", q, k, v, w.masked_fill(gone, low), bk, do, kvalid=kv, q_offset=off)
    check(got, reference("relpos", q, k, v, w.masked_fill(gone, -math.inf), bk, do=do, kvalid=kv, q_offset=off))
    assert not got["o"][:, :, 1].any() and bool((got["lse"][:, 1] == -math.inf).all()) and not got["dq"][:, :, 1].any() and not got["dw"][gone].any()


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("Sq, Sk", [(70, 100), (150, 200)])
@pytest.mark.parametrize("D", HEADS["relpos"])
def test_rows_at_a_large_negative_bias_stay_finite(D, Sq, Sk, t):
    """Head 0 has -1e9 at every position: its statistics are tens of units coarse, its gradients must be finite all the same, head 1 exact."""
    q, k, v, w, bk, do = make("relpos", TYPES[t], 2, 2, 2, D, Sq, Sk, buckets=8, reach=40)
    w[:, 0] = -1e9
    got = run("relpos", q, k, v, w, bk, do)
    for n, x in got.items():
        assert bool(torch.isfinite(x).all()), n
    assert got["o"][:, :, 0].abs().max() <= v[:, :, 0].abs().max()
    want = reference("relpos", q, k, v, w, bk, do=do)
    head1 = lambda n, x: x[:, 1] if n in ("lse", "dw") else x[:, :, 1]
    check({n: head1(n, x) for n, x in got.items()}, {n: tuple(head1(n, y) for y in want[n]) for n in got})


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_strides(op):
    """Views of a packed projection, head-major storage, a key shared over the batch, a slice of a longer cache, operands that have to be copied."""
    q, k, v, w, bk, do = make(op, torch.bfloat16, 2, 4, 4, 32, 90, 90, seed=18)
    want = run(op, q, k, v, w, bk, do)
    same = lambda got: all(torch.equal(got[n], want[n]) for n in got)
    width = [x[0, 0].numel() for x in (q, k, v)]
    packed = torch.cat([x.reshape(2, 90, -1) for x in (q, k, v)], 2)
    assert same(run(op, *(p.unflatten(2, x.shape[2:]) for p, x in zip(packed.split(width, 2), (q, k, v))), w, bk, do))
    major = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert same(run(op, *major, w, bk, do.transpose(1, 2).contiguous().transpose(1, 2)))
    cache = [torch.cat([x, x], 1)[:, :90] for x in (k, v)]
    assert same(run(op, q, *cache, w, bk, do))
    odd = [torch.cat([x, x[..., :1]], -1)[..., :-1] for x in (q, k, v)]              # rows of an odd number of elements
    assert same(run(op, *odd, w, bk, do))
    off = [torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape) for x in (q, k, v, do)]   # addresses off by one element
    assert same(run(op, *off[:3], w, bk, off[3]))
    shared = [x[:1].expand(x.shape) for x in (k, v)]
    got, ref = run(op, q, *shared, w, bk, do), run(op, q, *(x.contiguous() for x in shared), w, bk, do)
    assert all(torch.equal(got[n], ref[n]) for n in got)
    far = torch.empty(3 * ((1 << 26) + 8), dtype=torch.bfloat16, device="cuda").view(3, -1)[:, : q[0, 0].numel()].unflatten(1, q.shape[2:])[None]
    far.copy_(q[:1, :3])                                     # positions more than 2^26 elements apart
    got, ref = (run(op, x, k[:1], v[:1], w, bk, do[:1, :3]) for x in (far, q[:1, :3]))
    assert all(torch.equal(got[n], ref[n]) for n in got)
    m = mask("holes", 2, 180)
    got, ref = run(op, q, k, v, w, bk, do, kvalid=m[:, ::2]), run(op, q, k, v, w, bk, do, kvalid=m[:, ::2].contiguous().bool())
    assert all(torch.equal(got[n], ref[n]) for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_offsets_beyond_32_bits(op):
    """A cache whose rows lie more than 2^31 elements apart."""
    q, k, v, w, bk, do = make(op, torch.bfloat16, 2, 1, 1, 32, 2, 300, seed=19)
    big = torch.empty(600 * (4 << 20), dtype=torch.bfloat16, device="cuda").view(2, 300, 4 << 20)
    kk, vv = big[:, :, : k[0, 0].numel()].unflatten(2, k.shape[2:]), big[:, :, 1024: 1024 + v[0, 0].numel()].unflatten(2, v.shape[2:])
    kk.copy_(k), vv.copy_(v)
    assert kk.stride(0) + 299 * kk.stride(1) > 2 ** 31
    got, want = run(op, q, kk, vv, w, bk, do), run(op, q, k, v, w, bk, do)
    assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_results_are_reproducible_and_rows_independent(op):
    x = make(op, torch.bfloat16, 4, 4, 2, 64, 300, 310, seed=20)
    m = mask("prefix", 4, 310)
    a = run(op, *x, kvalid=m)
    for _ in range(3):
        b = run(op, *x, kvalid=m)
        assert all(torch.equal(a[n], b[n]) for n in a)
    q, k, v, w, bk, do = x                                   # a sample does not depend on its neighbours in the batch
    one = run(op, q[2:3], k[2:3], v[2:3], w, bk, do[2:3], kvalid=m[2:3])
    for n in ("o", "lse", "dq", "dk", "dv"):
        assert torch.equal(one[n][0], a[n][2]), n


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_autograd_and_forward_alone(op):
    from univtg_amd import attention
    q, k, v, w, bk, do = make(op, torch.bfloat16, 2, 4, 2, 32, 60, 75, seed=21)
    m = mask("prefix", 2, 75)
    f = (lambda *x: attention.relpos_attention(*x, bk, kvalid=m)) if op == "relpos" else (lambda *x: attention.diff_attention(*x, kvalid=m))
    want = run(op, q, k, v, w, bk, do, kvalid=m)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, w)]
    o = f(*leaves)
    o.backward(do)
    assert torch.equal(o, want["o"])
    for x, n in zip(leaves, ("dq", "dk", "dv", "dw")):
        assert torch.equal(x.grad, want[n]), n
    with torch.no_grad():
        assert torch.equal(f(*leaves), o) and not f(*leaves).requires_grad
    frozen = leaves[3].detach()                              # no gradient for the weights: theirs is not computed
    o = f(*leaves[:3], frozen)
    assert torch.equal(torch.autograd.grad(o, leaves[0], do)[0], want["dq"])
    wh = w.to(torch.bfloat16).requires_grad_(True)
    o = f(q, k, v, wh)
    assert torch.autograd.grad(o.float().sum(), wh)[0].dtype == torch.bfloat16
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(f(*leaves).float().sum(), leaves[0], create_graph=True)
        g.float().sum().backward()


@pytest.mark.gpu
def test_layers_together_train_and_serve():
    """An encoder block of each kind, one behind the other, trained and then served token by token against a cache: gradients of every parameter against
    autograd through the formulas in 64 bits, served rows against the whole pass."""
    from univtg_amd import attention, ops
    torch.manual_seed(3)
    B, S, H, D, W = 2, 70, 4, 32, 128
    bk = ops.relpos_buckets(16, 40, bidirectional=False)
    P = {"w1": torch.randn(W, 3 * W) * W ** -0.5, "w2": torch.randn(W, 5 * W) * W ** -0.5, "wo": torch.randn(2 * W, W) * (2 * W) ** -0.5,
         "table": torch.randn(16, H), "lam": torch.rand(H)}
    P = {n: x.cuda() for n, x in P.items()}
    x = torch.randn(B, S, W, device="cuda")
    m = torch.ones(B, S, dtype=torch.uint8, device="cuda")
    m[1, 50:] = 0

    def net(p, x, dt, kernels):
        q, k, v = (x @ p["w1"]).to(dt).view(B, S, 3, H, D).unbind(2)
        if kernels:
            a = attention.relpos_attention(q, k, v, p["table"], bk, kvalid=m, causal=True)
        else:
            a = plain("relpos", q, k, v, p["table"])
        y = (x + a.reshape(B, S, W).to(x.dtype)) @ p["w2"]
        z = y.to(dt)
        q, k, v = z[..., : 2 * W].unflatten(2, (H, 2, D)), z[..., 2 * W: 4 * W].unflatten(2, (H, 2, D)), z[..., 4 * W:].unflatten(2, (H, D))
        v = torch.cat([v, v], -1)
        if kernels:
            a2 = attention.diff_attention(q, k, v, p["lam"], kvalid=m, causal=True)
        else:
            a2 = plain("diff", q, k, v, p["lam"])
        return a2.reshape(B, S, 2 * W).to(x.dtype) @ p["wo"]

    hide = _hide(B, S, S, m, True, 0, "cuda")
    rel = (torch.arange(S, device="cuda")[None] - torch.arange(S, device="cuda")[:, None]).clamp(-40, 40) + 40

    def plain(op, q, k, v, w):
        t = lambda z: z.transpose(1, 2)
        if op == "relpos":
            s = t(q) @ t(k).transpose(2, 3) * D ** -0.5 + w[bk.long()[rel]].permute(2, 0, 1)
            return t(torch.softmax(s.masked_fill(hide, -math.inf), -1) @ t(v))
        a = [torch.softmax((t(q[:, :, :, i]) @ t(k[:, :, :, i]).transpose(2, 3) * D ** -0.5).masked_fill(hide, -math.inf), -1) for i in (0, 1)]
        return t((a[0] - w.view(1, H, 1, 1) * a[1]) @ t(v))

    gout = torch.randn(B, S, W, device="cuda")
    p32 = {n: z.clone().requires_grad_(True) for n, z in P.items()}
    p64 = {n: z.double().requires_grad_(True) for n, z in P.items()}
    y = net(p32, x, torch.float16, True)
    y.backward(gout)
    y64 = net(p64, x.double(), torch.float64, False)
    y64.backward(gout.double())
    # a chain of about eight roundings to 11 bits (q / k / v, p, o, ds of two layers) whose errors are independent from element to element: in the
    # 2-norm each adds at most u sqrt(3) of what it rounds, and differences of softmax maps are at most a few times smaller than their parts
    tol = 8 * math.sqrt(3) * 2.0 ** -11 * 4
    for a, b in [(y, y64)] + [(p32[n].grad, p64[n].grad) for n in P]:
        assert float((a.double() - b).norm() / b.norm()) < tol
    with torch.no_grad():                                    # serving: the first layer, one token at a time against the keys so far
        q, k, v = (x @ P["w1"]).half().view(B, S, 3, H, D).unbind(2)
        whole, _ = ops.relpos_attention_fwd(q, k, v, P["table"], bk, causal=True)
        ref = reference("relpos", q, k, v, P["table"], bk, causal=True)["o"]
        for i in (0, 1, 31, 32, 69):
            o, _ = ops.relpos_attention_fwd(q[:, i: i + 1], k[:, : i + 1], v[:, : i + 1], P["table"], bk, q_offset=i)
            assert ((o[:, 0].double() - ref[0][:, i]).abs() <= ref[1][:, i]).all() and ((o[:, 0] - whole[:, i]).double().abs() <= 2 * ref[1][:, i]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_streams_and_graphs(op):
    """Another stream than the default one, two calls in flight on two streams, and a captured forward and backward, replayed on new inputs."""
    x = make(op, torch.bfloat16, 2, 4, 2, 64, 100, 120, seed=22)
    y = make(op, torch.bfloat16, 2, 4, 2, 64, 100, 120, seed=23)
    z = make(op, torch.bfloat16, 1, 4, 2, 64, 1, 900, seed=24)
    wx, wy, wz = run(op, *x), run(op, *y), run(op, *z)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        gx, gz = run(op, *x), run(op, *z)
    with torch.cuda.stream(s2):
        gy = run(op, *y)
    torch.cuda.synchronize()
    for got, want in ((gx, wx), (gy, wy), (gz, wz)):
        assert all(torch.equal(got[n], want[n]) for n in got)
    static, sz = [t.clone() if t is not None else None for t in x], [t.clone() if t is not None else None for t in z]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run(op, *static), run(op, *sz)
    torch.cuda.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(op, *static)
    with torch.cuda.graph(graph2):
        outz = run(op, *sz)
    for src, want in ((y, wy), (x, wx), (y, wy)):
        for a, b in zip(static, src):
            if a is not None:
                a.copy_(b)
        graph.replay(), graph2.replay(), graph.replay()
        eager = run(op, *src)                                # the program's own work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(out[n], want[n]) and torch.equal(eager[n], want[n]) for n in out)
        assert all(torch.equal(outz[n], wz[n]) for n in outz)


@pytest.mark.gpu
def test_captured_training_step():
    """A training step captured into a graph.  While an eager graph of the same leaves is alive it is refused before anything is enqueued: autograd's
    engine would join the eager graph's stream to the capture, which ends the process."""
    from univtg_amd import attention
    q, k, v, w, _, do = make("diff", torch.bfloat16, 1, 2, 2, 32, 40, 40, seed=25)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, w)]
    alive = attention.diff_attention(*leaves)
    want = torch.autograd.grad(attention.diff_attention(*leaves), leaves, do)
    own = [t.detach().requires_grad_(True) for t in leaves]
    refused = 0
    for x in (own, leaves):
        if x is leaves:
            with pytest.raises(RuntimeError, match="still holds a leaf"):
                attention._check_capture(leaves, torch.cuda.Stream().cuda_stream)
            refused += 1
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, leaves, do), want))
            del alive                                        # the last eager graph of these leaves: now they may be captured
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = torch.autograd.grad(attention.diff_attention(*x), x, do)
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert refused == 1


@pytest.mark.gpu
def test_refusals_name_the_argument():
    from univtg_amd import ops
    q, k, v, w, bk, do = make("relpos", torch.bfloat16, 1, 2, 2, 32, 4, 6)
    o, lse = ops.relpos_attention_fwd(q, k, v, w, bk)
    cases = [
        (ValueError, "shapes", lambda: ops.relpos_attention_fwd(q, k[:, :5], v, w, bk)),
        (ValueError, "q and k must be", lambda: ops.relpos_attention_fwd(q[0], k, v, w, bk)),
        (ValueError, "bfloat16 or all float16", lambda: ops.relpos_attention_fwd(q.float(), k.float(), v.float(), w, bk)),
        (ValueError, "bfloat16 or all float16", lambda: ops.relpos_attention_fwd(q, k.half(), v, w, bk)),
        (ValueError, "kvalid", lambda: ops.relpos_attention_fwd(q, k, v, w, bk, kvalid=torch.ones(1, 6, device="cuda"))),
        (ValueError, "kvalid", lambda: ops.relpos_attention_fwd(q, k, v, w, bk, kvalid=torch.ones(1, 4, dtype=torch.uint8, device="cuda"))),
        (ValueError, "must be on", lambda: ops.relpos_attention_fwd(q, k.cpu(), v, w, bk)),
        (ValueError, "table", lambda: ops.relpos_attention_fwd(q, k, v, w[:, :1], bk)),
        (ValueError, "table", lambda: ops.relpos_attention_fwd(q, k, v, w.cpu(), bk)),
        (ValueError, "buckets", lambda: ops.relpos_attention_fwd(q, k, v, w, bk[:-1])),
        (ValueError, "buckets", lambda: ops.relpos_attention_fwd(q, k, v, w, bk.long())),
        (RuntimeError, "scale", lambda: ops.relpos_attention_fwd(q, k, v, w, bk, scale=-1.0)),
        (ValueError, "q_offset", lambda: ops.relpos_attention_fwd(q, k, v, w, bk, q_offset=1 << 32, causal=True)),
        (RuntimeError, "head_dim", lambda: ops.relpos_attention_fwd(q[..., :16], k[..., :16], v[..., :16], w, bk)),
        (RuntimeError, "H must be", lambda: ops.relpos_attention_fwd(q, k.repeat(1, 1, 2, 1)[:, :, :3], v.repeat(1, 1, 2, 1)[:, :, :3], w, bk)),
        (RuntimeError, "non-positive", lambda: ops.relpos_attention_fwd(q[:, :0], k, v, w, bk)),
        (RuntimeError, "reach", lambda: ops.relpos_attention_fwd(q, k, v, w, bk[:1])),
        (ValueError, "do and o", lambda: ops.relpos_attention_bwd(do[:, :2], q, k, v, w, bk, o, lse)),
        (ValueError, "do must be", lambda: ops.relpos_attention_bwd(do.float(), q, k, v, w, bk, o, lse)),
        (ValueError, "do must be", lambda: ops.relpos_attention_bwd(do.cpu(), q, k, v, w, bk, o, lse)),
        (ValueError, "o must be", lambda: ops.relpos_attention_bwd(do, q, k, v, w, bk, o.cpu(), lse)),
        (ValueError, "lse must be", lambda: ops.relpos_attention_bwd(do, q, k, v, w, bk, o, lse.cpu())),
        (ValueError, "lse must be", lambda: ops.relpos_attention_bwd(do, q, k, v, w, bk, o, lse.double())),
    ]
    q2, k2, v2, lam, _, do2 = make("diff", torch.float16, 1, 2, 2, 64, 4, 6)
    od, lse2, o2 = ops.diff_attention_fwd(q2, k2, v2, lam, need_o2=True)
    cases += [
        (ValueError, "shapes", lambda: ops.diff_attention_fwd(q2[:, :, :, :1], k2, v2, lam)),
        (ValueError, "shapes", lambda: ops.diff_attention_fwd(q2, k2, v2[..., :64], lam)),
        (ValueError, "lam", lambda: ops.diff_attention_fwd(q2, k2, v2, lam[:1])),
        (RuntimeError, "32 or 64", lambda: ops.diff_attention_fwd(torch.cat([q2, q2], -1), torch.cat([k2, k2], -1), torch.cat([v2, v2], -1), lam)),
        (ValueError, "do, o and o2", lambda: ops.diff_attention_bwd(do2, q2, k2, v2, lam, od, o2[:, :2], lse2)),
        (ValueError, "o2 must be", lambda: ops.diff_attention_bwd(do2, q2, k2, v2, lam, od, o2.cpu(), lse2)),
        (ValueError, "lse must be", lambda: ops.diff_attention_bwd(do2, q2, k2, v2, lam, od, o2, lse2.cpu())),
    ]
    for kind, text, call in cases:
        with pytest.raises(kind, match=text):
            call()
