"""What the attention cores' autograd layer relies on between a forward and a backward call.  Saved-tensor hooks (activation offloading, compression) may
hand the backward call equal values in another layout than the forward call laid out; other derivatives than the first ones in reverse mode are refused.
Workgroups that stay leave reserved compute units alone.  On the CPU the library is a stand-in that notes its arguments."""
import pytest
import torch


class Library:
    """Takes every call, computes nothing, keeps the descriptor and the tensors behind the addresses."""
    def __init__(self, monkeypatch):
        from univtg_amd import _lib, ops
        self.calls, self.tensors, at = [], {}, ops._at
        monkeypatch.setattr(_lib, "load", lambda: self)
        monkeypatch.setattr(ops, "_elsewhere", lambda t: False)
        monkeypatch.setattr(ops, "_stream_of", lambda t: 0)
        monkeypatch.setattr(ops, "_at", lambda t: None if t is None else self.tensors.setdefault(at(t), t).data_ptr())

    def uvtg_attn_ws_bytes(self, d, maps, backward):
        return 0

    def __getattr__(self, name):
        if not name.startswith("uvtg_"):
            raise AttributeError(name)

        def call(d, *args):
            self.calls.append((name, {n: getattr(d, n) for n, _ in d._fields_}, [self.tensors.get(a) for a in args]))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    return Library(monkeypatch)


def packed(op, B, S, H, D, dev, t=torch.bfloat16):
    """q, k, v as views of one projection, which is how an encoder layer has them."""
    g = torch.Generator(device=dev).manual_seed(4)
    if op == "relpos":
        return torch.randn(B, S, 3, H, D, generator=g, device=dev).to(t).unbind(2)
    x = torch.randn(B, S, 3, 2 * H * D, generator=g, device=dev).to(t)
    return [x[:, :, 0].unflatten(2, (H, 2, D)), x[:, :, 1].unflatten(2, (H, 2, D)), x[:, :, 2].unflatten(2, (H, 2 * D))]


def weights(op, H, dev):
    from univtg_amd import ops
    if op == "relpos":
        return torch.linspace(-1, 1, 8 * H, device=dev).view(8, H), ops.relpos_buckets(8, 20, device=dev)
    return torch.linspace(0.1, 0.8, H, device=dev), None


def attend(op, q, k, v, w, buckets, **opts):
    from univtg_amd import attention
    return attention.relpos_attention(q, k, v, w, buckets, **opts) if op == "relpos" else attention.diff_attention(q, k, v, w, **opts)


RELAYOUTS = {
    "dense": lambda t: t.clone(memory_format=torch.contiguous_format),                                   # what torch.autograd.graph.save_on_cpu returns
    "unaligned": lambda t: torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape),
    "axes": lambda t: t.permute(*range(t.dim())[::-1]).contiguous().permute(*range(t.dim())[::-1]),
    "halves": lambda t: torch.stack([t, t], 0)[0] if t.dim() < 2 else torch.stack([t, t], 1)[:, 0],      # samples twice as far apart
    "strided": lambda t: torch.stack([t, t], -1)[..., 0],
}


@pytest.mark.parametrize("how", RELAYOUTS)
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_backward_describes_the_operands_it_is_given(library, op, how):
    B, S, H, D = 2, 10, 4, 32
    q, k, v = packed(op, B, S, H, D, "cpu")
    w, bk = weights(op, H, "cpu")
    kvalid = (torch.arange(S) < 7).to(torch.uint8).expand(B, S)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, w)]
    assert leaves[0].stride(1) == 3 * H * D * (2 if op == "diff" else 1)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: RELAYOUTS[how](t.detach())):
        o = attend(op, *leaves, bk, kvalid=kvalid)
        o.backward(torch.ones_like(o))
    (_, _, fwd), (name, d, bwd) = library.calls
    assert name.endswith("attention_bwd")
    n = 6 if op == "relpos" else 5                           # q, k, v, table and buckets or lam, kvalid
    for a, b in zip(fwd[:n], bwd[:n]):
        assert torch.equal(a, b)
    for x, prefix, axes in ((bwd[0], "q", "bshm"), (bwd[1], "k", "bshm"), (bwd[2], "v", "bsh")):
        assert x.data_ptr() % 16 == 0 and x.stride(-1) == 1
        for axis, stride in zip(axes, x.stride()[:-1]):
            assert d[f"{prefix}_s{axis}"] == stride and stride % 8 == 0, (prefix, axis)
    assert bwd[n - 1].stride() == (d["kvalid_sb"], 1)
    saved = bwd[3: n - 1] + bwd[n: n + (3 if op == "relpos" else 4)]                                     # weights; o, (o2,) lse, dO
    assert all(x.is_contiguous() and x.data_ptr() % 4 == 0 for x in saved) and all(x.data_ptr() % 16 == 0 for x in saved if x.dim() == 4 and x.dtype == q.dtype)


@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_forward_mode_is_refused(library, op):
    """A tangent of an operand, or of the gradient that comes in, would be lost."""
    from torch.autograd import forward_ad
    q, k, v = packed(op, 2, 10, 4, 32, "cpu")
    w, bk = weights(op, 4, "cpu")
    with forward_ad.dual_level():
        for i in range(4):
            x = [q, k, v, w]
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    attend(op, *x, bk)
        attend(op, q, k, v, w, bk)                           # (no tangent: as ever)
        leaf = q.detach().requires_grad_(True)
        o = attend(op, leaf, k, v, w, bk)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(o, leaf, forward_ad.make_dual(torch.ones_like(o), torch.ones_like(o)))


@pytest.mark.gpu
@pytest.mark.parametrize("how", RELAYOUTS)
@pytest.mark.parametrize("op", ["relpos", "diff"])
def test_gradients_do_not_depend_on_saved_tensor_hooks(op, how):
    """Short rows and longer ones (one kernel, two passes), packed views, a mask shared over the batch."""
    for S, H, D in ((70, 4, 32), (150, 2, 64)):
        q, k, v = packed(op, 2, S, H, D, "cuda")
        w, bk = weights(op, H, "cuda")
        kvalid = (torch.arange(S, device="cuda") < S - 9).to(torch.uint8).expand(2, S)
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, w)]
        do = torch.randn(2, S, H, v.shape[-1], device="cuda").to(q.dtype)
        want = torch.autograd.grad(attend(op, *leaves, bk, kvalid=kvalid), leaves, do)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: RELAYOUTS[how](t.detach())):
            got = torch.autograd.grad(attend(op, *leaves, bk, kvalid=kvalid), leaves, do)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with torch.autograd.graph.save_on_cpu():
            got = torch.autograd.grad(attend(op, *leaves, bk, kvalid=kvalid), leaves, do)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("op, D", [("relpos", 128), ("diff", 32), ("relpos", 32)])
def test_reserved_compute_units_stay_free(op, D):
    """The backward of short rows keeps its workgroups: with all but 8 compute units reserved (of 256) it runs on those 8 alone, at least 4 times as long,
    and gives the same bits."""
    from test_attention_maps import make
    from univtg_amd import _lib, ops
    q, k, v, w, bk, do = make(op, torch.bfloat16, 128, 8, 8, D, 64, 64)
    if op == "relpos":
        o, lse = ops.relpos_attention_fwd(q, k, v, w, bk)
        bwd = lambda: ops.relpos_attention_bwd(do, q, k, v, w, bk, o, lse)
    else:
        o, lse, o2 = ops.diff_attention_fwd(q, k, v, w, need_o2=True)
        bwd = lambda: ops.diff_attention_bwd(do, q, k, v, w, o, o2, lse)

    def timed():
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        bwd()
        ev[0].record()
        for _ in range(5):
            out = bwd()
        ev[1].record()
        torch.cuda.synchronize()
        return ev[0].elapsed_time(ev[1]), out
    lib = _lib.load()
    whole, want = timed()
    try:
        assert lib.uvtg_set_reserved_cus(1 << 16) == 8
        few, got = timed()
    finally:
        lib.uvtg_set_reserved_cus(0)
    assert few > 4 * whole and all(torch.equal(a, b) for a, b in zip(got, want))
