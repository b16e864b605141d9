"""Calls of the decoder operators at the edge of what their documentation allows: saved tensors that come back in another layout, sizes and types at
the end of their range, derivatives that do not exist, gradients far from one."""
import pytest
import torch

from las_pytorch_amd import _cabi, cross_attention
from las_pytorch_amd.model import cross_attention as ca
from las_pytorch_amd.solver import solver as S


class Recorder:
    """Stands where the library call stands, on the CPU: keeps each call's descriptor and addresses, computes nothing."""

    def __init__(self, monkeypatch):
        self.calls = []
        monkeypatch.setattr(ca, "_refuse", lambda *operands: None)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
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


def _keep_all(monkeypatch, alive):
    """Every tensor that .contiguous() or .clone() gives stays alive (what is freed could come back at the address of another)."""
    keep = lambda f: lambda x, *a, **k: (alive.append(f(x, *a, **k)), alive[-1])[1]      # noqa: E731
    monkeypatch.setattr(torch.Tensor, "contiguous", keep(torch.Tensor.contiguous))
    monkeypatch.setattr(torch.Tensor, "clone", keep(torch.Tensor.clone))


def _held_at(address, like, strides, alive):
    """The values that a kernel reads at ``address`` by ``strides``, none of them outside the storage that lies there."""
    (held,) = {id(x): x for x in alive if x.data_ptr() == address and x.shape == like.shape}.values()
    last = held.storage_offset() + sum((n - 1) * s for n, s in zip(like.shape, strides))
    assert last < held.untyped_storage().nbytes() // held.element_size(), (strides, held.stride())
    return held.as_strided(like.shape, strides)


@pytest.mark.parametrize("how", ["dense", "permuted", "between"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["fused", "time first", "heads first", "plain"])
def test_backward_addresses_the_tensors_that_arrive(monkeypatch, layout, dtype, how):
    """The descriptor of the backward's call against the storage behind its addresses: every row where the tensor has it, none outside."""
    recorder = Recorder(monkeypatch)
    leaves = [x.detach().requires_grad_(True) for x in _views(dtype, "cpu")[layout]]
    lengths = torch.tensor([45, 0, 7], dtype=torch.int32)
    alive = []
    with torch.autograd.graph.saved_tensors_hooks(lambda x: _moved(x, how), lambda x: (alive.append(x), x)[1]):
        out = cross_attention(*leaves, lengths)
    _keep_all(monkeypatch, alive)
    torch.autograd.grad(out, leaves, torch.ones_like(out))
    monkeypatch.undo()
    forward, backward = recorder.calls
    d, addresses = backward[0], backward[1:8]
    assert (d.B, d.U, d.T, d.H, d.Hkv, d.D, d.scale) == tuple(getattr(forward[0], n) for n in ("B", "U", "T", "H", "Hkv", "D", "scale"))
    want = {0: (leaves[0], (d.q_b, d.q_u, d.q_h)), 1: (leaves[1], (d.k_b, d.k_t, d.k_h)), 2: (leaves[2], (d.v_b, d.v_t, d.v_h))}
    for i, (leaf, strides) in want.items():
        assert addresses[i] % 16 == 0
        assert torch.equal(_held_at(addresses[i], leaf, (*strides, 1), alive), leaf), (i, strides)
    for i in (3, 4, 5):                                 # lengths, the output, its statistics: contiguous
        assert any(x.data_ptr() == addresses[i] and x.is_contiguous() for x in alive)
    assert addresses[4] % 16 == 0


@pytest.mark.parametrize("how", ["dense", "permuted", "between"])
@pytest.mark.parametrize("seed", [1.0, 2.0])
@pytest.mark.parametrize("layout", ["plain", "step first", "padded"])
def test_distillation_backward_addresses_the_tensors_that_arrive(monkeypatch, layout, seed, how):
    """The same of the distillation loss, whose first backward hands over what the forward formed and whose second forms it anew."""
    recorder = Recorder(monkeypatch)
    g = torch.Generator().manual_seed(33)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    z = {"plain": r(3, 5, 40), "step first": r(5, 3, 40).transpose(0, 1), "padded": r(3, 5, 48)[..., :40]}[layout].requires_grad_(True)
    index, teacher, lengths = torch.randint(0, 40, (3, 5, 4), generator=g), r(3, 5, 4), torch.tensor([5, 0, 2], dtype=torch.int32)
    alive = []
    with torch.autograd.graph.saved_tensors_hooks(lambda x: _moved(x, how), lambda x: (alive.append(x), x)[1]):
        loss = S._DistillationLoss.apply(z, index, teacher, lengths, 2.0)
    _keep_all(monkeypatch, alive)
    for keep in (True, False):
        torch.autograd.grad(loss, (z,), torch.tensor(seed), retain_graph=keep)
    monkeypatch.undo()
    for d, *addresses in recorder.calls[1:]:
        assert (d.B, d.U, d.V, d.K) == (3, 5, 40, 4)
        assert torch.equal(_held_at(addresses[0], z, (d.stride_b, d.stride_u, 1), alive), z)
        for at, like in zip(addresses[1:], (index, teacher, lengths)):
            assert torch.equal(_held_at(at, like, torch.empty(like.shape).stride(), alive), like)


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
