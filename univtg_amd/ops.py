"""Thin tensor-level wrappers over the kernel-level entry points of include/uvtg.h (the same kernels the
engine launches).  Used by the parity tests and handy for experiments; no computation happens in Python."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .model import _f32c, _ptr, _stream


def _need_cuda(t):
    if not t.is_cuda:
        raise RuntimeError("univtg_amd.ops: tensors must be on a ROCm device (no CPU fallback)")


def to_bf16_bits(x: torch.Tensor) -> torch.Tensor:
    """fp32 -> bf16 (round-to-nearest-even) on device, returned as torch.bfloat16."""
    _need_cuda(x)
    x = _f32c(x)
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    _lib.check(_lib.load().uvtg_cast_bf16(_ptr(x), _ptr(out), x.numel(), _stream()), "uvtg_cast_bf16")
    return out


def sk_workspace(device) -> torch.Tensor:
    """Split-K workspace of the small-launch GEMM entry points (tickets zeroed; include/uvtg.h: uvtg_linear_*_sk)."""
    return torch.zeros(int(_lib.load().uvtg_linear_sk_ws_floats()), device=device)


def linear_bf16(a_bf16, w_bf16, bias=None, act=0, sk_ws=None):
    """C = act(A W^T + b): A [M,K] bf16, W [N,K] bf16 -> fp32 [M,N].  sk_ws (sk_workspace()): small launches may split K."""
    _need_cuda(a_bf16)
    M, K = a_bf16.shape
    N = w_bf16.shape[0]
    out = torch.empty(M, N, device=a_bf16.device)
    if sk_ws is not None:
        _lib.check(_lib.load().uvtg_linear_bf16_sk(_ptr(a_bf16.contiguous()), _ptr(w_bf16.contiguous()), _ptr(bias), _ptr(out),
                                                   M, N, K, act, _ptr(sk_ws), _stream()), "uvtg_linear_bf16_sk")
        return out
    _lib.check(_lib.load().uvtg_linear_bf16(_ptr(a_bf16.contiguous()), _ptr(w_bf16.contiguous()), _ptr(bias), _ptr(out),
                                            M, N, K, act, _stream()), "uvtg_linear_bf16")
    return out


def split_f16(x, is_weight=False):
    """fp16 hi | lo operand images [rows, 2 * kp] of an fp32 matrix (kp = columns rounded up to 64); see include/uvtg.h."""
    _need_cuda(x)
    x = _f32c(x)
    rows, cols = x.shape
    kp = (cols + 63) // 64 * 64
    out = torch.empty(rows, 2 * kp, dtype=torch.float16, device=x.device)
    _lib.check(_lib.load().uvtg_split_f16(_ptr(x), _ptr(out), rows, cols, kp, int(is_weight), _stream()), "uvtg_split_f16")
    return out


def linear_f32x3(a, w, bias=None, act=0, sk_ws=None):
    """nn.Linear in the precise arithmetic: fp32 operands -> fp16 hi | lo images -> three-product split GEMM (uvtg_linear_split)."""
    _need_cuda(a)
    a, w = _f32c(a), _f32c(w)
    M, K = a.shape
    N = w.shape[0]
    sa, sw = split_f16(a, False), split_f16(w, True)
    out = torch.empty(M, N, device=a.device)
    if sk_ws is not None:
        _lib.check(_lib.load().uvtg_linear_split_sk(_ptr(sa), _ptr(sw), _ptr(bias), _ptr(out), M, N, sa.shape[1] // 2, act, _ptr(sk_ws), _stream()),
                   "uvtg_linear_split_sk")
        return out
    _lib.check(_lib.load().uvtg_linear_split(_ptr(sa), _ptr(sw), _ptr(bias), _ptr(out), M, N, sa.shape[1] // 2, act, _stream()), "uvtg_linear_split")
    return out


def wgrad_bf16(dy_bf16, x_bf16, splits=4, with_bias=True):
    """dW [N,K] = dY^T X, db [N] = colsum(dY)."""
    _need_cuda(dy_bf16)
    M, N = dy_bf16.shape
    K = x_bf16.shape[1]
    dw = torch.zeros(N, K, device=dy_bf16.device)
    db = torch.zeros(N, device=dy_bf16.device) if with_bias else None
    _lib.check(_lib.load().uvtg_wgrad_bf16(_ptr(dy_bf16.contiguous()), _ptr(x_bf16.contiguous()), _ptr(dw), _ptr(db),
                                           M, N, K, splits, _stream()), "uvtg_wgrad_bf16")
    return dw, db


def wgrad_bf16_ws(dy_bf16, x_bf16, with_bias=True):
    """Same as wgrad_bf16 with the scratch that enables the 256-tile slab + reduce kernel."""
    _need_cuda(dy_bf16)
    lib = _lib.load()
    M, N = dy_bf16.shape
    K = x_bf16.shape[1]
    dw = torch.zeros(N, K, device=dy_bf16.device)
    db = torch.zeros(N, device=dy_bf16.device) if with_bias else None
    nf = lib.uvtg_wgrad_scratch_floats(M, N, K)
    scratch = torch.empty(nf, device=dy_bf16.device)
    _lib.check(lib.uvtg_wgrad_bf16_ws(_ptr(dy_bf16.contiguous()), _ptr(x_bf16.contiguous()), _ptr(dw), _ptr(db), M, N, K,
                                      _ptr(scratch), nf, _stream()), "uvtg_wgrad_bf16_ws")
    return dw, db


def wgrad_bf16_multi(dys, xs, with_bias=True):
    """Several weight gradients over the same rows in one launch, no reduce pass (uvtg_wgrad_bf16_multi).  dys[i] [M, N_i], xs[i] [M, K_i]
    bf16-bit tensors; returns ([dW_i], [dbias_i])."""
    lib = _lib.load()
    _need_cuda(dys[0])
    n = len(dys)
    M = dys[0].shape[0]
    dev = dys[0].device
    Ns, Ks = [int(t.shape[1]) for t in dys], [int(t.shape[1]) for t in xs]
    tiles = sum((a // 256) * (b // 256) for a, b in zip(Ns, Ks))
    nf = lib.uvtg_wgrad_multi_slab_floats(tiles)
    slabs = torch.empty(nf, device=dev)
    tickets = torch.zeros(tiles, dtype=torch.int32, device=dev)
    dws = [torch.full((a, b), float("nan"), device=dev) for a, b in zip(Ns, Ks)]       # assigned: every element must be written
    dbs = [torch.zeros(a, device=dev) for a in Ns] if with_bias else None
    arr = lambda ts: (C.c_void_p * n)(*[t.data_ptr() for t in ts])
    iarr = lambda vs: (C.c_int * n)(*vs)
    _lib.check(lib.uvtg_wgrad_bf16_multi(n, arr(dys), iarr(Ns), arr(xs), iarr(Ks), arr(dws), arr(dbs) if with_bias else None, M,
                                         _ptr(slabs), nf, _ptr(tickets), tiles, _stream()), "uvtg_wgrad_bf16_multi")
    return dws, dbs


def layernorm_fwd(x, gamma, beta):
    _need_cuda(x)
    x = _f32c(x)
    rows, D = x.shape
    y = torch.empty_like(x)
    mean = torch.empty(rows, device=x.device)
    rstd = torch.empty(rows, device=x.device)
    _lib.check(_lib.load().uvtg_layernorm_fwd(_ptr(x), _ptr(_f32c(gamma)), _ptr(_f32c(beta)), _ptr(y), _ptr(mean), _ptr(rstd),
                                              rows, D, _stream()), "uvtg_layernorm_fwd")
    return y, mean, rstd


def layernorm_bwd(g, x, mean, rstd, gamma):
    _need_cuda(x)
    rows, D = x.shape
    dx = torch.empty_like(x)
    dgamma = torch.zeros(D, device=x.device)
    dbeta = torch.zeros(D, device=x.device)
    _lib.check(_lib.load().uvtg_layernorm_bwd(_ptr(_f32c(g)), _ptr(_f32c(x)), _ptr(mean), _ptr(rstd), _ptr(_f32c(gamma)),
                                              _ptr(dx), _ptr(dgamma), _ptr(dbeta), rows, D, _stream()), "uvtg_layernorm_bwd")
    return dx, dgamma, dbeta


def attention_fwd(qkv, kvalid, B, S, H, hd, precise=False):
    """qkv [B*S, 3*H*hd] (bf16, or fp32 when precise; q already scaled), kvalid [B,S] uint8 -> o [B*S, H*hd], lse [B,H,S]."""
    _need_cuda(qkv)
    o = torch.empty(B * S, H * hd, dtype=qkv.dtype, device=qkv.device)
    lse = torch.empty(B, H, S, device=qkv.device)
    _lib.check(_lib.load().uvtg_attention_fwd(_ptr(qkv.contiguous()), _ptr(kvalid.contiguous()), _ptr(o), _ptr(lse),
                                              B, S, H, hd, int(precise), _stream()), "uvtg_attention_fwd")
    return o, lse


def attention_bwd(qkv, kvalid, o, lse, do, qscale, B, S, H, hd):
    _need_cuda(qkv)
    dqkv = torch.zeros_like(qkv)
    delta = torch.empty(B, H, S, device=qkv.device)
    _lib.check(_lib.load().uvtg_attention_bwd(_ptr(qkv.contiguous()), _ptr(kvalid.contiguous()), _ptr(o.contiguous()), _ptr(lse),
                                              _ptr(do.contiguous()), _ptr(delta), _ptr(dqkv), float(qscale), B, S, H, hd, _stream()),
               "uvtg_attention_bwd")
    return dqkv


def sine_position(vid_mask, txt_mask, dim_t):
    _need_cuda(vid_mask)
    B, Lv = vid_mask.shape
    Lt = txt_mask.shape[1]
    d = dim_t.numel()
    pos = torch.empty(B, Lv, d, device=vid_mask.device)
    kvalid = torch.empty(B, Lv + Lt, dtype=torch.uint8, device=vid_mask.device)
    _lib.check(_lib.load().uvtg_sine_position(_ptr(_f32c(vid_mask)), _ptr(_f32c(txt_mask)), _ptr(_f32c(dim_t)), _ptr(pos), _ptr(kvalid),
                                              B, Lv, Lt, d, _stream()), "uvtg_sine_position")
    return pos, kvalid


def decode_rank_nms(pred_logits, pred_spans, timestamp, timestamp_mask, durations, nms_thd=0.7, max_before=1000, max_after=10):
    """Device version of main/inference_mr.py:109-160 + utils/temporal_nms.py.  Returns (windows [B,Lv,3] float64 ranked
    rows, order [B,Lv] int32 clip index per rank, keep [B,max_after] int32 ranked positions kept (-1 pad), n_keep [B])."""
    _need_cuda(pred_logits)
    B, Lv = pred_logits.shape[:2]
    dev = pred_logits.device
    win = torch.empty(B, Lv, 3, dtype=torch.float64, device=dev)
    order = torch.empty(B, Lv, dtype=torch.int32, device=dev)
    keep = torch.empty(B, max_after, dtype=torch.int32, device=dev)
    nk = torch.empty(B, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().uvtg_decode_rank_nms(_ptr(_f32c(pred_logits)), _ptr(_f32c(pred_spans)), _ptr(_f32c(timestamp)),
                                                _ptr(_f32c(timestamp_mask)), _ptr(_f32c(durations)), B, Lv, float(nms_thd),
                                                int(max_before), int(max_after), _ptr(win), _ptr(order), _ptr(keep), _ptr(nk),
                                                _stream()), "uvtg_decode_rank_nms")
    return win, order, keep, nk


def postprocess_mr(pred_logits, pred_spans, saliency, timestamp, timestamp_mask, durations, clip_length=0.0, eval_mode="add",
                   nms_thd=0.7, max_before=1000, max_after=10):
    """decode_rank_nms + PostProcessorDETR round_multiple (clip_length > 0) before the NMS + pred_saliency_scores
    (fp16(saliency) [+ prob]); main/inference_mr.py:109-192, eval/postprocessing.py:46-51.  Returns
    (windows, order, keep, n_keep, saliency_out[B,Lv] fp32 or None)."""
    _need_cuda(pred_logits)
    B, Lv = pred_logits.shape[:2]
    dev = pred_logits.device
    win = torch.empty(B, Lv, 3, dtype=torch.float64, device=dev)
    order = torch.empty(B, Lv, dtype=torch.int32, device=dev)
    keep = torch.empty(B, max_after, dtype=torch.int32, device=dev)
    nk = torch.empty(B, dtype=torch.int32, device=dev)
    sal_out = torch.empty(B, Lv, device=dev) if saliency is not None else None
    _lib.check(_lib.load().uvtg_postprocess_mr(_ptr(_f32c(pred_logits)), _ptr(_f32c(pred_spans)), _ptr(None if saliency is None else _f32c(saliency)),
                                               _ptr(_f32c(timestamp)), _ptr(_f32c(timestamp_mask)), _ptr(_f32c(durations)), B, Lv,
                                               float(clip_length), int(eval_mode == "add"), float(nms_thd), int(max_before), int(max_after),
                                               _ptr(win), _ptr(order), _ptr(keep), _ptr(nk), _ptr(sal_out), _stream()), "uvtg_postprocess_mr")
    return win, order, keep, nk, sal_out


# ---- attention over score maps: learned relative position bias by buckets, differential heads -------------------------------------------
_ATTN_TYPES = {torch.bfloat16: 0, torch.float16: 1}


def relpos_buckets(num_buckets, max_distance, bidirectional=True, device="cuda"):
    """Bucket of every relative position (key minus query) -max_distance .. max_distance, int32 [2 * max_distance + 1]: the lower half of the
    buckets holds one distance each, the upper half is spaced evenly in the logarithm up to max_distance, from where on the last one holds all.
    bidirectional: half of the buckets for keys behind the query (and at it), half for keys ahead; else keys ahead share bucket 0.
    Borders are found in whole numbers, so that none depends on how a logarithm is rounded."""
    n = num_buckets // 2 if bidirectional else num_buckets
    exact = n // 2
    if n < 2 or (bidirectional and num_buckets % 2) or max_distance <= exact:
        raise ValueError(f"relpos_buckets: {num_buckets} buckets cannot be spaced up to a distance of {max_distance}")
    steps, b, behind = n - exact, 0, []
    for d in range(max_distance + 1):
        if d < exact:
            behind.append(d)
            continue
        # bucket exact + b from (d / exact) ** steps >= (max_distance / exact) ** b on
        while b < steps - 1 and d ** steps * exact ** (b + 1) >= max_distance ** (b + 1) * exact ** steps:
            b += 1
        behind.append(exact + b)
    ahead = [n + b for b in behind[1:]] if bidirectional else [behind[0]] * max_distance
    return torch.tensor(behind[::-1] + ahead, dtype=torch.int32, device=device)


def _attn_operand(t):
    """t as the kernels address it and its strides: channels contiguous, every other stride and the address a multiple of 16 bytes, positions at most
    2^26 elements apart (else a contiguous copy); the stride of an axis of one entry is never used."""
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0:
        if (st[0] | st[1] | st[2] | (st[3] if len(st) == 5 else 0)) & 7 == 0 and st[1] <= 1 << 26:
            return t, st
        st = [s if n > 1 else 0 for n, s in zip(t.shape[:-1], st)]
        if all(s % 8 == 0 for s in st) and st[1] <= 1 << 26:
            return t, st
    t = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
    return t, t.stride()


def _attn_call(name, maps, q, k, v, kvalid, q_offset, causal, scale):
    """Checks and lays out the operands both attentions share: (dims, q, k, v, kvalid)."""
    qs, ks, vs, dtype, dev = q.shape, k.shape, v.shape, q.dtype, q.device
    if len(qs) != 3 + maps or len(ks) != 3 + maps or len(vs) != 4:
        raise ValueError(f"{name}: q and k must be [B, S, heads, {'2, ' if maps == 2 else ''}D] and v [B, Sk, Hkv, {'2 D' if maps == 2 else 'D'}]")
    B, Sq, H, D, Sk, Hkv = qs[0], qs[1], qs[2], qs[-1], ks[1], ks[2]
    if (maps == 2 and (qs[3] != 2 or ks[3] != 2)) or ks[0] != B or ks[-1] != D or vs != (B, Sk, Hkv, maps * D):
        raise ValueError(f"{name}: shapes do not agree: q {tuple(qs)}, k {tuple(ks)}, v {tuple(vs)}")
    if dtype not in _ATTN_TYPES or k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"{name}: q, k and v must all be bfloat16 or all float16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if k.device != dev or v.device != dev or (kvalid is not None and kvalid.device != dev):
        raise ValueError(f"{name}: every operand must be on {dev}")
    q, qs = _attn_operand(q)
    k, ks = _attn_operand(k)
    v, vs = _attn_operand(v)
    mask_sb = 0
    if kvalid is not None:
        if kvalid.dtype not in (torch.uint8, torch.bool) or kvalid.shape != (B, Sk):
            raise ValueError(f"{name}: kvalid must be uint8 or bool [B, Sk] = [{B}, {Sk}], got {kvalid.dtype} {tuple(kvalid.shape)}")
        if kvalid.stride(1) != 1:
            kvalid = kvalid.contiguous()
        mask_sb = kvalid.stride(0)
    if not -(1 << 28) <= q_offset <= 1 << 28:
        raise ValueError(f"{name}: q_offset must lie within +-2^28, got {q_offset}")
    d = _lib.AttnDims(0, _ATTN_TYPES[dtype], B, H, Hkv, D, Sq, Sk, 1 if causal else 0, int(q_offset), D ** -0.5 if scale is None else float(scale), 0, 0,
                      qs[0], qs[1], qs[2], qs[3] if maps == 2 else 0, ks[0], ks[1], ks[2], ks[3] if maps == 2 else 0, vs[0], vs[1], vs[2], mask_sb)
    d.layout = (qs, ks, vs)
    return d, q, k, v, kvalid


def _attn_unchanged(d, q, k, v, kvalid, dense):
    """Whether operands that autograd kept since their call laid them out are still laid out that way (`dense`: those that are contiguous).  Saved-tensor
    hooks (offloading, compression) return equal values in whatever layout."""
    dev, address = q.get_device(), q.data_ptr() | k.data_ptr() | v.data_ptr()
    if (q.stride(), k.stride(), v.stride()) != d.layout or k.get_device() != dev or v.get_device() != dev or not q.dtype == k.dtype == v.dtype:
        return False
    if kvalid is not None and (kvalid.stride() != (d.kvalid_sb, 1) or kvalid.get_device() != dev):
        return False
    for t in dense:
        if not t.is_contiguous() or t.get_device() != dev:
            return False
        address |= t.data_ptr()
    return not address & 15


def _attn_ws(lib, d, maps, backward, like):
    n = lib.uvtg_attn_ws_bytes(d, maps, backward)
    return like.new_empty(n, dtype=torch.uint8) if n else None


def _elsewhere(t):
    """Whether t is on another GPU than the current one, whose streams the call would then use."""
    _need_cuda(t)
    return t.device.index != torch.cuda.current_device()


def _stream_of(t):
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _relpos_operands(d, q, table, buckets):
    if table.dim() != 2 or table.shape[1] != d.H or table.device != q.device:
        raise ValueError(f"relpos_attention: table must be [n_buckets, H = {d.H}] on {q.device}, got {tuple(table.shape)} on {table.device}")
    if buckets.dim() != 1 or buckets.dtype != torch.int32 or buckets.numel() % 2 == 0 or buckets.device != q.device:
        raise ValueError(f"relpos_attention: buckets must be int32 [2 * reach + 1] on {q.device}, got {buckets.dtype} {tuple(buckets.shape)} on {buckets.device}")
    d.n_buckets, d.reach = table.shape[0], buckets.numel() // 2
    return _f32c(table), buckets.contiguous()


def _attn_saved(name, t, like, what, dtype=None):
    if t.dtype != (dtype or like.dtype) or t.device != like.device:
        raise ValueError(f"{name}: {what} must be {dtype or like.dtype} on {like.device}")
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _at(t):
    return None if t is None else t.data_ptr()


def _relpos_fwd(q, k, v, table, buckets, kvalid, q_offset, causal, scale):
    """(o, lse) and what the backward call reads again: the descriptor and the operands as laid out."""
    lib = _lib.load()
    d, q, k, v, kvalid = _attn_call("relpos_attention", 1, q, k, v, kvalid, q_offset, causal, scale)
    table, buckets = _relpos_operands(d, q, table, buckets)
    o = q.new_empty((d.B, d.Sq, d.H, d.D))
    lse = q.new_empty((d.B, d.H, d.Sq), dtype=torch.float32)
    ws = _attn_ws(lib, d, 1, 0, q)
    _lib.check(lib.uvtg_relpos_attention_fwd(d, _at(q), _at(k), _at(v), _at(table), _at(buckets), _at(kvalid), _at(o), _at(lse), _at(ws), _stream_of(q)),
               "uvtg_relpos_attention_fwd")
    return o, lse, (d, q, k, v, table, buckets, kvalid)


def _relpos_bwd(do, d, q, k, v, table, buckets, kvalid, o, lse, need_dtable):
    lib = _lib.load()
    if not _attn_unchanged(d, q, k, v, kvalid, (table, buckets, o, lse)):
        d, q, k, v, kvalid = _attn_call("relpos_attention_bwd", 1, q, k, v, kvalid, d.q_offset, d.causal, d.scale)
        table, buckets = _relpos_operands(d, q, table, buckets)
        o, lse = _attn_saved("relpos_attention_bwd", o, q, "o"), _attn_saved("relpos_attention_bwd", lse, q, "lse", torch.float32)
    do = _attn_saved("relpos_attention_bwd", do, q, "do")
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    dtable = table.new_empty(table.shape) if need_dtable else None
    ws = _attn_ws(lib, d, 1, 1, q)
    _lib.check(lib.uvtg_relpos_attention_bwd(d, _at(q), _at(k), _at(v), _at(table), _at(buckets), _at(kvalid), _at(o), _at(lse), _at(do), _at(dq), _at(dk),
                                             _at(dv), _at(dtable), _at(ws), _stream_of(q)), "uvtg_relpos_attention_bwd")
    return dq, dk, dv, dtable


def relpos_attention_fwd(q, k, v, table, buckets, kvalid=None, q_offset=0, causal=False, scale=None):
    """softmax(scale q k^T + table[buckets[clamp(j - i - q_offset)], h]) v: q [B, Sq, H, D], k and v [B, Sk, Hkv, D] (bf16 or fp16, D 32 / 64 / 128,
    any strides), table [n_buckets, H] fp32, buckets int32 [2 reach + 1] (relpos_buckets), kvalid [B, Sk] uint8 / bool (0 = masked key).  causal:
    query i sees keys up to i + q_offset; k and v rows that are masked, or behind what any query sees, may hold anything.  A table entry of -inf takes its
    positions out of the row.  scale defaults to D ** -0.5.  Returns o [B, Sq, H, D] and lse [B, H, Sq] (fp32); a row that sees no key is 0 with lse -inf."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return relpos_attention_fwd(q, k, v, table, buckets, kvalid, q_offset, causal, scale)
    return _relpos_fwd(q, k, v, table, buckets, kvalid, q_offset, causal, scale)[:2]


def relpos_attention_bwd(do, q, k, v, table, buckets, o, lse, kvalid=None, q_offset=0, causal=False, scale=None, need_dtable=True):
    """Gradients of relpos_attention_fwd from its outputs and do: dq, dk, dv (the operands' type, contiguous) and dtable (fp32, or None: its last sums are
    left out then, not its workspace of 4 bytes per position within reach, 16 keys, head and sample)."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return relpos_attention_bwd(do, q, k, v, table, buckets, o, lse, kvalid, q_offset, causal, scale, need_dtable)
    d, q, k, v, kvalid = _attn_call("relpos_attention", 1, q, k, v, kvalid, q_offset, causal, scale)
    table, buckets = _relpos_operands(d, q, table, buckets)
    if do.shape != (d.B, d.Sq, d.H, d.D) or o.shape != do.shape or lse.shape != (d.B, d.H, d.Sq):
        raise ValueError("relpos_attention_bwd: do and o must be [B, Sq, H, D], lse [B, H, Sq]")
    return _relpos_bwd(do, d, q, k, v, table, buckets, kvalid, _attn_saved("relpos_attention_bwd", o, q, "o"),
                       _attn_saved("relpos_attention_bwd", lse, q, "lse", torch.float32), need_dtable)


def _lam_operand(d, q, lam):
    if lam.shape != (d.H,) or lam.device != q.device:
        raise ValueError(f"diff_attention: lam must be [H = {d.H}] on {q.device}, got {tuple(lam.shape)} on {lam.device}")
    return _f32c(lam)


def _diff_fwd(q, k, v, lam, kvalid, q_offset, causal, scale, need_o2):
    lib = _lib.load()
    d, q, k, v, kvalid = _attn_call("diff_attention", 2, q, k, v, kvalid, q_offset, causal, scale)
    lam = _lam_operand(d, q, lam)
    o = q.new_empty((d.B, d.Sq, d.H, 2 * d.D))
    o2 = torch.empty_like(o) if need_o2 else None
    lse = q.new_empty((d.B, d.H, 2, d.Sq), dtype=torch.float32)
    ws = _attn_ws(lib, d, 2, 0, q)
    _lib.check(lib.uvtg_diff_attention_fwd(d, _at(q), _at(k), _at(v), _at(lam), _at(kvalid), _at(o), _at(o2), _at(lse), _at(ws), _stream_of(q)),
               "uvtg_diff_attention_fwd")
    return o, lse, o2, (d, q, k, v, lam, kvalid)


def _diff_bwd(do, d, q, k, v, lam, kvalid, o, o2, lse, need_dlam):
    lib = _lib.load()
    if not _attn_unchanged(d, q, k, v, kvalid, (lam, o, o2, lse)):
        d, q, k, v, kvalid = _attn_call("diff_attention_bwd", 2, q, k, v, kvalid, d.q_offset, d.causal, d.scale)
        lam = _lam_operand(d, q, lam)
        o, o2 = _attn_saved("diff_attention_bwd", o, q, "o"), _attn_saved("diff_attention_bwd", o2, q, "o2")
        lse = _attn_saved("diff_attention_bwd", lse, q, "lse", torch.float32)
    do = _attn_saved("diff_attention_bwd", do, q, "do")
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    dlam = lam.new_empty(d.H) if need_dlam else None
    ws = _attn_ws(lib, d, 2, 1, q)
    _lib.check(lib.uvtg_diff_attention_bwd(d, _at(q), _at(k), _at(v), _at(lam), _at(kvalid), _at(o), _at(o2), _at(lse), _at(do), _at(dq), _at(dk), _at(dv),
                                           _at(dlam), _at(ws), _stream_of(q)), "uvtg_diff_attention_bwd")
    return dq, dk, dv, dlam


def diff_attention_fwd(q, k, v, lam, kvalid=None, q_offset=0, causal=False, scale=None, need_o2=False):
    """Differential attention (softmax(scale q1 k1^T) - lam[h] softmax(scale q2 k2^T)) v: q [B, Sq, H, 2, D], k [B, Sk, Hkv, 2, D], v [B, Sk, Hkv, 2 D]
    (bf16 or fp16, D 32 / 64, any strides), lam [H] fp32; kvalid, q_offset, causal and scale as in relpos_attention_fwd.  Returns o [B, Sq, H, 2 D]
    and lse [B, H, 2, Sq] (fp32), and with need_o2 also o2, the second map's own output, which the backward pass reads."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return diff_attention_fwd(q, k, v, lam, kvalid, q_offset, causal, scale, need_o2)
    o, lse, o2, _ = _diff_fwd(q, k, v, lam, kvalid, q_offset, causal, scale, need_o2)
    return (o, lse, o2) if need_o2 else (o, lse)


def diff_attention_bwd(do, q, k, v, lam, o, o2, lse, kvalid=None, q_offset=0, causal=False, scale=None, need_dlam=True):
    """Gradients of diff_attention_fwd(need_o2=True) from its outputs and do: dq, dk, dv (the operands' type, contiguous) and dlam (fp32, or None)."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return diff_attention_bwd(do, q, k, v, lam, o, o2, lse, kvalid, q_offset, causal, scale, need_dlam)
    d, q, k, v, kvalid = _attn_call("diff_attention", 2, q, k, v, kvalid, q_offset, causal, scale)
    lam = _lam_operand(d, q, lam)
    if do.shape != (d.B, d.Sq, d.H, 2 * d.D) or o.shape != do.shape or o2.shape != do.shape or lse.shape != (d.B, d.H, 2, d.Sq):
        raise ValueError("diff_attention_bwd: do, o and o2 must be [B, Sq, H, 2 D], lse [B, H, 2, Sq]")
    o, o2 = (_attn_saved("diff_attention_bwd", t, q, w) for t, w in ((o, "o"), (o2, "o2")))
    return _diff_bwd(do, d, q, k, v, lam, kvalid, o, o2, _attn_saved("diff_attention_bwd", lse, q, "lse", torch.float32), need_dlam)
