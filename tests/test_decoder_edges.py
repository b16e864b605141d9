"""Calls of the decoder operators at the edge of what their documentation allows: saved tensors that come back in another layout, sizes and types at
the end of their range, derivatives that do not exist, gradients far from one."""
import pytest
import torch

from las_pytorch_amd import _cabi, cross_attention
from las_pytorch_amd.model import cross_attention as ca


class Recorder:
    """Stands where the library call stands, on the CPU: keeps each call's descriptor and addresses, computes nothing."""

    def __init__(self, monkeypatch):
        self.calls = []
        monkeypatch.setattr(ca, "_refuse", lambda *operands: None)
        monkeypatch.setattr(_cabi, "call_on", lambda device, fn, *args: self.calls.append(args))


def _moved(x, how):
    """The values of ``x`` as a hook may hand them back: dense, in another order of its dimensions, or between 16-byte pieces."""
    if how == "dense":
        return x.clone(memory_format=torch.contiguous_format)
    if how == "permuted":
        order = list(range(x.dim()))[::-1]
        return x.permute(order).contiguous().permute(order)
    return torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape).copy_(x)


def _views(dtype, device, seed=31):
    """(query, key, value) as programs hold them: a fused key / value projection, time first, and plain."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)      # noqa: E731
    B, U, T, H, Hkv, D = 3, 21, 45, 4, 2, 64
    kv = r(B, T, 2, Hkv, D)
    return {"fused": (r(B, U, H, D), kv[:, :, 0], kv[:, :, 1]),
            "time first": (r(U, B, H, D).transpose(0, 1), r(T, B, Hkv, D).transpose(0, 1), r(B, T, Hkv, D)),
            "heads first": tuple(r(B, h, n, D).transpose(1, 2) for h, n in ((H, U), (Hkv, T), (Hkv, T))),
            "plain": (r(B, U, H, D), r(B, T, Hkv, D), r(B, T, Hkv, D))}


@pytest.mark.parametrize("how", ["dense", "permuted", "between"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["fused", "time first", "heads first", "plain"])
def test_backward_addresses_the_tensors_that_arrive(monkeypatch, layout, dtype, how):
    """The descriptor of the backward's call against the storage behind its addresses: every row where the tensor has it, none outside."""
    recorder = Recorder(monkeypatch)
    leaves = [x.detach().requires_grad_(True) for x in _views(dtype, "cpu")[layout]]
    lengths = torch.tensor([45, 0, 7], dtype=torch.int32)
    alive = []                                          # (what is freed could come back at the address of another)
    contiguous, clone = torch.Tensor.contiguous, torch.Tensor.clone
    keep = lambda f: lambda x, *a, **k: (alive.append(f(x, *a, **k)), alive[-1])[1]      # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(lambda x: _moved(x, how), lambda x: (alive.append(x), x)[1]):
        out = cross_attention(*leaves, lengths)
    monkeypatch.setattr(torch.Tensor, "contiguous", keep(contiguous))
    monkeypatch.setattr(torch.Tensor, "clone", keep(clone))
    torch.autograd.grad(out, leaves, torch.ones_like(out))
    monkeypatch.undo()
    forward, backward = recorder.calls
    d, addresses = backward[0], backward[1:8]
    assert (d.B, d.U, d.T, d.H, d.Hkv, d.D, d.scale) == tuple(getattr(forward[0], n) for n in ("B", "U", "T", "H", "Hkv", "D", "scale"))
    want = {0: (leaves[0], (d.q_b, d.q_u, d.q_h)), 1: (leaves[1], (d.k_b, d.k_t, d.k_h)), 2: (leaves[2], (d.v_b, d.v_t, d.v_h))}
    for i, (leaf, strides) in want.items():
        assert addresses[i] % 16 == 0
        (held,) = {id(x): x for x in alive if x.data_ptr() == addresses[i] and x.shape == leaf.shape}.values()
        last = held.storage_offset() + sum((n - 1) * s for n, s in zip(leaf.shape, (*strides, 1)))
        assert last < held.untyped_storage().nbytes() // held.element_size(), (i, strides, held.stride())
        assert torch.equal(held.as_strided(leaf.shape, (*strides, 1)), leaf), (i, strides, held.stride())
    for i in (3, 4, 5):                                 # lengths, the output, its statistics: contiguous
        assert any(x.data_ptr() == addresses[i] and x.is_contiguous() for x in alive)
    assert addresses[4] % 16 == 0


@pytest.mark.gpu
@pytest.mark.parametrize("pinned", [False, True], ids=["plain", "pinned"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", ["fused", "time first", "heads first", "plain"])
def test_views_whose_saved_tensors_are_kept_on_the_host(layout, dtype, pinned):
    """Views that come back from the host in another layout: the bits of the backward that kept them."""
    leaves = [x.detach().requires_grad_(True) for x in _views(dtype, "cuda")[layout]]
    lengths = torch.tensor([45, 0, 7], dtype=torch.int32, device="cuda")
    dout = torch.randn(3, 21, 4, 64, generator=torch.Generator().manual_seed(32)).to(dtype).cuda()
    want = torch.autograd.grad(cross_attention(*leaves, lengths), leaves, dout)
    with torch.autograd.graph.save_on_cpu(pin_memory=pinned):
        out = cross_attention(*leaves, lengths)
    for a, b in zip(torch.autograd.grad(out, leaves, dout), want):
        assert torch.equal(a, b)
