"""Cases of the attention operators that stand beside the masked attention core: attention with a learned relative position bias by buckets
(`relpos`) and differential attention (`diff`), each as a training step (forward and all gradients) and as a serving call (forward alone, whole
prompts, chunks of a few tokens and single tokens against a long cache).

    relpos   o = softmax(scale q k^T + table[bucket(j - i - q_offset)]) v
    diff     o = softmax(scale q1 k1^T) v - lam softmax(scale q2 k2^T) v

`run` computes them with elementary operations in 32 bits, or, where `own` is true, with the framework's kernels."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- the cases --------------------------------------------------------------------------------------------------------------------------
def _case(name, op, mode, dtype, B, H, Hkv, D, Sq, Sk, causal, fill, buckets=32, reach=128):
    c = dict(name=name, op=op, mode=mode, dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, Sq=Sq, Sk=Sk, causal=causal, fill=fill)
    return dict(c, buckets=buckets, reach=reach) if op == "relpos" else c


def listed():
    return [
        # one new token of one stream against a short history: the latency of a call
        _case("relpos one token", "relpos", "fwd", "bf16", 1, 8, 8, 128, 1, 257, True, 1.0),
        # the clip + text tokens of a training batch (75 + 32 positions, padded samples), width 1024
        _case("relpos encoder step", "relpos", "train", "bf16", 256, 8, 8, 128, 107, 107, False, 0.5),
        # the same encoder on long videos (1200 clips + 32 text tokens)
        _case("relpos long video step", "relpos", "train", "bf16", 32, 8, 8, 128, 1232, 1232, False, 0.5),
        # queries of one length over a memory of another (text over clips), small heads, half precision
        _case("relpos cross step", "relpos", "train", "fp16", 24, 12, 12, 32, 333, 601, False, 0.3, 48, 400),
        # one long causal prompt, shared key / value heads
        _case("relpos prompt", "relpos", "fwd", "fp16", 2, 16, 4, 64, 8191, 8191, True, 1.0, 64, 512),
        # single tokens of a batch of streams against a long cache
        _case("relpos long cache", "relpos", "fwd", "bf16", 16, 16, 4, 128, 1, 32765, True, 0.7),
        # one new token of one stream, differential heads
        _case("diff one token", "diff", "fwd", "bf16", 1, 8, 8, 64, 1, 300, True, 1.0),
        # the encoder's training batch with differential heads of the same width (2 x 64 per head)
        _case("diff encoder step", "diff", "train", "bf16", 256, 8, 8, 64, 107, 107, False, 0.5),
        # a causal training step over long rows with shared key / value heads
        _case("diff causal step", "diff", "train", "bf16", 4, 16, 4, 64, 4096, 4096, True, 1.0),
        # small heads, half precision, an odd length
        _case("diff small heads step", "diff", "train", "fp16", 8, 12, 12, 32, 1501, 1501, False, 0.6),
        # an encoder pass over a very long video, no gradients
        _case("diff long video", "diff", "fwd", "bf16", 2, 8, 8, 64, 6007, 6007, False, 0.9),
        # a few new tokens of a batch of streams against a long cache
        _case("diff long cache", "diff", "fwd", "fp16", 16, 16, 4, 64, 5, 20011, True, 0.7),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["relpos", "diff"])
        mode = rng.choice(["train", "train", "fwd", "cache"])
        D = rng.choice([32, 64, 128] if op == "relpos" else [32, 64])
        Hkv = rng.choice([1, 2, 4, 8, 12])
        H = Hkv * rng.choice([1, 1, 1, 2, 4])
        B = _spread(rng, 1, 256)
        causal = rng.random() < 0.5
        if mode == "cache":
            Sk = _spread(rng, 64, 60000)
            Sq = min(Sk, rng.choice([1, 1, 1, rng.randint(2, 64)]))
        else:
            Sk = _spread(rng, 16, 8192)
            Sq = Sk if rng.random() < 0.6 else _spread(rng, 16, 8192)
            causal = causal and Sq <= Sk
        c = _case("", op, "train" if mode == "train" else "fwd", rng.choice(["bf16", "fp16"]), B, H, Hkv, D, Sq, Sk, causal,
                  rng.choice([1.0, round(rng.uniform(0.2, 0.95), 2)]), rng.choice([16, 32, 64]), _spread(rng, 64, 1024))
        del c["name"]
        w = work(c)
        # (score matrices of the plain form at most about 16 GB, caches at most about 8 GB)
        if w["flops"] <= most and w["bytes"] <= 8e9 and w["flops"] >= 1e5 and B * H * Sq * Sk <= 4 << 30:
            return c


def _pairs(c):
    """(query, key) pairs of one head that are not masked, on average over the lengths that `prepare` draws."""
    keys = c["Sk"] * (1.0 + c["fill"]) / 2
    if not c["causal"]:
        return c["B"] * c["Sq"] * keys
    return c["B"] * c["Sq"] * min(keys, c["Sk"] - (c["Sq"] - 1) / 2)


def work(case):
    c = case
    maps, dv = (2, 2 * c["D"]) if c["op"] == "diff" else (1, c["D"])
    fill = (1.0 + c["fill"]) / 2
    q, o = c["B"] * c["Sq"] * c["H"] * maps * c["D"], c["B"] * c["Sq"] * c["H"] * dv
    kv = c["B"] * c["Sk"] * c["Hkv"] * (maps * c["D"] + dv)
    pairs = _pairs(c) * c["H"]
    if c["mode"] == "fwd":
        # q, valid k / v, o in 16 bits and the row statistics; the scores of each map and one product with v
        return {"bytes": 2 * (q + kv * fill + o) + 4 * c["B"] * c["Sq"] * c["H"] * maps, "flops": 2 * pairs * (maps * c["D"] + dv)}
    # forward, then scores, dP, dV, dQ and dK of every map; q, k, v, dO in, o and the gradients out
    return {"bytes": 2 * (2 * q + kv * fill + kv + 2 * o), "flops": 2 * pairs * (4 * maps * c["D"] + 3 * dv)}


# ---- inputs -----------------------------------------------------------------------------------------------------------------------------
def _bucket(d, n, reach):
    """Bucket 0 .. n - 1 of a distance d >= 0: the lower half exactly, the upper half spaced evenly in the logarithm up to `reach`, in whole numbers."""
    e = n // 2
    if d < e:
        return d
    m, b = n - e, 0
    # largest b with (d / e)^m >= (reach / e)^b
    while b < m - 1 and d ** m * e ** (b + 1) >= reach ** (b + 1) * e ** m:
        b += 1
    return e + b


def _bucket_map(n, reach, causal):
    """Bucket of each relative position -reach .. reach (key minus query): halves for keys behind and ahead, or all of them for keys behind."""
    if causal:
        behind = [_bucket(d, n, reach) for d in range(reach + 1)]
        return behind[:0:-1] + [behind[0]] * (reach + 1)
    half = [_bucket(d, n // 2, reach) for d in range(reach + 1)]
    return half[:0:-1] + [half[0]] + [n // 2 + b for b in half[1:]]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[c["dtype"]]
    B, Sq, Sk, H, Hkv, D = (c[k] for k in ("B", "Sq", "Sk", "H", "Hkv", "D"))
    train = c["mode"] == "train"

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32) * std).to(dtype)

    s = {"case": dict(c), "scale": D ** -0.5, "q_offset": Sk - Sq if c["causal"] else 0, "causal": c["causal"], "kvalid": None}
    maps = (2,) if c["op"] == "diff" else ()
    if Sq == Sk and H == Hkv and c["op"] == "relpos":       # one packed projection, as the encoder's: strided views
        qkv = normal(B, Sk, 3, H, D)
        q, k, v = qkv.unbind(2)
    else:
        q, k = normal(B, Sq, H, *maps, D), normal(B, Sk, Hkv, *maps, D)
        v = normal(B, Sk, Hkv, 2 * D if maps else D)
    if c["fill"] < 1:
        least = max(1, int(c["fill"] * Sk))
        lens = torch.randint(least, Sk + 1, (B, 1), generator=gen, device=DEV)
        if c["causal"]:                                      # a stream's newest token sees its whole history
            lens[0] = Sk
        s["kvalid"] = (torch.arange(Sk, device=DEV)[None] < lens).to(torch.uint8)
    if c["op"] == "relpos":
        s["table"] = normal(c["buckets"], H, std=0.5, dtype=torch.float32)
        s["buckets"] = torch.tensor(_bucket_map(c["buckets"], c["reach"], c["causal"]), dtype=torch.int32, device=DEV)
    else:
        s["lam"] = torch.rand(H, generator=gen, device=DEV) * 0.7 + 0.1
    s["q"], s["k"], s["v"] = q, k, v
    if train:
        s["do"] = normal(B, Sq, H, 2 * D if maps else D)
        for n in ("q", "k", "v", "table", "lam"):
            if n in s:
                s[n] = s[n].detach().requires_grad_(True)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    opts = dict(kvalid=s["kvalid"], q_offset=s["q_offset"], causal=s["causal"], scale=s["scale"])
    if "do" not in s:
        from univtg_amd import ops
        if "table" in s:
            o, lse = ops.relpos_attention_fwd(s["q"], s["k"], s["v"], s["table"], s["buckets"], **opts)
        else:
            o, lse = ops.diff_attention_fwd(s["q"], s["k"], s["v"], s["lam"], **opts)
        return {"o": o, "lse": lse}
    from univtg_amd import attention
    if "table" in s:
        o = attention.relpos_attention(s["q"], s["k"], s["v"], s["table"], s["buckets"], **opts)
        dq, dk, dv, dtable = torch.autograd.grad(o, (s["q"], s["k"], s["v"], s["table"]), s["do"])
        return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}
    o = attention.diff_attention(s["q"], s["k"], s["v"], s["lam"], **opts)
    dq, dk, dv, dlam = torch.autograd.grad(o, (s["q"], s["k"], s["v"], s["lam"]), s["do"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def _masked(s):
    """Truth values [B or 1, 1, Sq or 1, Sk] of the positions that a query must not see, or None."""
    c, off = None, s["q_offset"]
    Sq, Sk = s["case"]["Sq"], s["case"]["Sk"]
    if s["causal"]:
        c = (torch.arange(Sk, device=DEV)[None] > torch.arange(Sq, device=DEV)[:, None] + off)[None, None]
    if s["kvalid"] is not None:
        pad = (s["kvalid"] == 0)[:, None, None]
        c = pad if c is None else c | pad
    return c


def _relative(s):
    """Index into the bucket map of every (query, key) pair: [Sq, Sk]."""
    Sq, Sk, R = s["case"]["Sq"], s["case"]["Sk"], s["case"]["reach"]
    rel = torch.arange(Sk, device=DEV)[None] - torch.arange(Sq, device=DEV)[:, None] - s["q_offset"]
    return rel.clamp(-R, R) + R


def _heads(x, H):
    """[B, S, h, d] in 16 bits -> [B, H, S, d] in 32, the shared heads repeated."""
    return x.detach().float().transpose(1, 2).repeat_interleave(H // x.shape[2], 1)


def _shared(x, Hkv, t):
    """[B, H, S, d] gradients -> [B, S, Hkv, d], summed over the heads that share one, rounded."""
    B, H, S, d = x.shape
    return x.view(B, Hkv, H // Hkv, S, d).sum(2).transpose(1, 2).to(t).contiguous()


def _softmax(x, mask):
    if mask is not None:
        x = x.masked_fill(mask, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    lse = (torch.log(total) + m)[..., 0]
    return p / torch.where(total == 0, torch.ones_like(total), total), lse


def _run_plain(s):
    c = s["case"]
    H, Hkv, t = c["H"], c["Hkv"], TYPES[c["dtype"]]
    mask, scale = _masked(s), s["scale"]
    v = _heads(s["v"], H)
    do = s["do"].float().transpose(1, 2) if "do" in s else None
    if "table" in s:
        q, k = _heads(s["q"], H), _heads(s["k"], H)
        idx = s["buckets"].long()[_relative(s)]
        p, lse = _softmax(torch.matmul(q, k.transpose(2, 3)) * scale + s["table"].detach()[idx].permute(2, 0, 1)[None], mask)
        o = torch.matmul(p, v).transpose(1, 2).to(t)
        if do is None:
            return {"o": o, "lse": lse}
        dv = torch.matmul(p.transpose(2, 3), do)
        dp = torch.matmul(do, v.transpose(2, 3))
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        dq = torch.matmul(ds, k) * scale
        dk = torch.matmul(ds.transpose(2, 3), q) * scale
        # the table's gradient: sums along the diagonals of the batch's sum, then over the diagonals of a bucket
        Sq, Sk, R = c["Sq"], c["Sk"], c["reach"]
        x = torch.nn.functional.pad(ds.sum(0).flip(1), (0, Sq)).reshape(H, -1)[:, : Sq * (Sk + Sq - 1)].view(H, Sq, Sk + Sq - 1)
        diag = x.sum(1, dtype=torch.float64)                 # relative position (key - query) -(Sq - 1) .. Sk - 1
        at = (torch.arange(Sk + Sq - 1, device=DEV) - (Sq - 1) - s["q_offset"]).clamp(-R, R) + R
        dtable = torch.zeros(c["buckets"], H, dtype=torch.float64, device=DEV).index_add_(0, s["buckets"].long()[at], diag.t().contiguous())
        return {"o": o, "dq": dq.transpose(1, 2).to(t), "dk": _shared(dk, Hkv, t), "dv": _shared(dv, Hkv, t), "dtable": dtable.float()}
    q1, q2 = _heads(s["q"][:, :, :, 0], H), _heads(s["q"][:, :, :, 1], H)
    k1, k2 = _heads(s["k"][:, :, :, 0], H), _heads(s["k"][:, :, :, 1], H)
    lam = s["lam"].detach()[None, :, None, None]
    p1, l1 = _softmax(torch.matmul(q1, k1.transpose(2, 3)) * scale, mask)
    p2, l2 = _softmax(torch.matmul(q2, k2.transpose(2, 3)) * scale, mask)
    p = p1 - lam * p2
    o = torch.matmul(p, v).transpose(1, 2).to(t)
    if do is None:
        return {"o": o, "lse": torch.stack([l1, l2], 2)}
    dv = torch.matmul(p.transpose(2, 3), do)
    dp = torch.matmul(do, v.transpose(2, 3))
    r1, r2 = (p1 * dp).sum(-1, keepdim=True), (p2 * dp).sum(-1, keepdim=True)
    ds1, ds2 = p1 * (dp - r1), -lam * p2 * (dp - r2)
    dq = torch.stack([torch.matmul(ds1, k1), torch.matmul(ds2, k2)], 3) * scale                  # [B, H, Sq, 2, D]
    dk1 = _shared(torch.matmul(ds1.transpose(2, 3), q1) * scale, Hkv, t)
    dk2 = _shared(torch.matmul(ds2.transpose(2, 3), q2) * scale, Hkv, t)
    dlam = -r2.double().sum((0, 2, 3))
    return {"o": o, "dq": dq.transpose(1, 2).to(t), "dk": torch.stack([dk1, dk2], 3), "dv": _shared(dv, Hkv, t), "dlam": dlam.float()}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    B, Sq, Sk, H, Hkv, D = (c[k] for k in ("B", "Sq", "Sk", "H", "Hkv", "D"))
    if B * H > 8192:
        return None
    G, train, diff = H // Hkv, "do" in s, c["op"] == "diff"
    f64 = dict(dtype=torch.float64, device=DEV)
    out = {"o": torch.zeros(B, Sq, H, 2 * D if diff else D, **f64)}
    if train:
        out |= {"dq": torch.zeros(s["q"].shape, **f64), "dk": torch.zeros(s["k"].shape, **f64), "dv": torch.zeros(s["v"].shape, **f64)}
    else:
        out["lse"] = torch.zeros((B, H, 2, Sq) if diff else (B, H, Sq), **f64)
    i, j = torch.arange(Sq, device=DEV)[:, None] + s["q_offset"], torch.arange(Sk, device=DEV)[None]
    late = (j > i) if s["causal"] else torch.zeros(Sq, Sk, dtype=torch.bool, device=DEV)
    if diff:
        out_w, weights = torch.zeros(H, **f64), s["lam"].detach().double()
    else:
        rel = (j - i).clamp(-c["reach"], c["reach"]) + c["reach"]
        bucket = s["buckets"].long()[rel]
        out_w, weights = torch.zeros(c["buckets"], H, **f64), s["table"].detach().double()
    del i, j
    with torch.enable_grad():
        for b in range(B):
            hide = late if s["kvalid"] is None else late | (s["kvalid"][b] == 0)[None]
            for h in range(H):
                n = h // G
                q = s["q"][b, :, h].detach().double().requires_grad_(train)
                k = s["k"][b, :, n].detach().double().requires_grad_(train)
                v = s["v"][b, :, n].detach().double().requires_grad_(train)
                if diff:
                    x = [q[:, m] @ k[:, m].t() * s["scale"] for m in (0, 1)]
                    w = weights[h].clone().requires_grad_(train)
                else:
                    w = weights[:, h][bucket].requires_grad_(train)
                    x = [q @ k.t() * s["scale"] + w]
                x = [t.masked_fill(hide, -math.inf) for t in x]
                p = [torch.softmax(t, -1) for t in x]
                o = (p[0] - w * p[1]) @ v if diff else p[0] @ v
                out["o"][b, :, h] = o.detach()
                if not train:
                    for m, t in enumerate(x):
                        (out["lse"][b, h, m] if diff else out["lse"][b, h]).copy_(torch.logsumexp(t, -1))
                    continue
                gq, gk, gv, gw = torch.autograd.grad(o, (q, k, v, w), s["do"][b, :, h].double())
                out["dq"][b, :, h] = gq
                out["dk"][b, :, n] += gk
                out["dv"][b, :, n] += gv
                if diff:
                    out_w[h] += gw
                else:
                    out_w[:, h] += torch.bincount(bucket.reshape(-1), gw.reshape(-1), minlength=c["buckets"])
    if train:
        out["dlam" if diff else "dtable"] = out_w
    return out
