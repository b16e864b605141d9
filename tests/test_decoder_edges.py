"""Calls of the decoder operators at the edge of what their documentation allows: saved tensors that come back in another layout, sizes and types at
the end of their range, derivatives that do not exist, gradients far from one."""
import math

import pytest
import torch

from las_pytorch_amd import _cabi, cross_attention, sample_tokens
from las_pytorch_amd.model import cross_attention as ca
from las_pytorch_amd.model.sampling import _limit
from las_pytorch_amd.solver import solver as S
from test_cross_attention import _check, _inputs
from test_sampling import _check as _check_draws


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


@pytest.mark.parametrize("between", [False, True], ids=["aligned", "between"])
def test_strides_of_dimensions_of_one(monkeypatch, between):
    """The stride of a dimension of one says nothing: one utterance out of a buffer whose rows are no whole 16-byte pieces, beside keys that start between them."""
    recorder = Recorder(monkeypatch)
    g = torch.Generator().manual_seed(40)
    q = torch.randn(3, 5 * 4 * 32 + 1, generator=g)[:, :-1].view(3, 5, 4, 32)[:1]
    k = torch.randn(9 * 2 * 32 + 1, generator=g)[1:] if between else torch.randn(9 * 2 * 32, generator=g)
    k = k.view(1, 9, 2, 32)
    assert q.stride(0) % 4 == 1 and (k.data_ptr() % 16 != 0) == between
    leaves = [x.detach().requires_grad_(True) for x in (q, k, k)]
    out = cross_attention(*leaves)
    torch.autograd.grad(out, leaves, torch.ones_like(out))
    for d, *addresses in recorder.calls:
        strides = [getattr(d, n) for n in ("q_b", "q_u", "q_h", "k_b", "k_t", "k_h", "v_b", "v_t", "v_h")]
        assert not any(s % 4 for s in strides), strides          # (what the library refuses)
        assert (d.q_u, d.q_h, d.k_t, d.k_h, d.v_t, d.v_h) == (128, 32, 64, 32, 64, 32)
        assert not any(a % 16 for a in addresses[:3])


def _with_tangents(*operands):
    """One operand after the other as a dual tensor."""
    for i, x in enumerate(operands):
        yield [*operands[:i], torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), *operands[i + 1:]]


def test_forward_mode_is_refused_before_the_call(monkeypatch):
    recorder = Recorder(monkeypatch)
    operands = _views(torch.float32, "cpu")["plain"]
    with torch.autograd.forward_ad.dual_level():
        for duals in _with_tangents(*operands):
            with pytest.raises(RuntimeError, match="forward-mode"):
                cross_attention(*duals)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                cross_attention(*duals)
        assert not recorder.calls
        cross_attention(*operands)                      # (no tangent: nothing to lose)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda q: cross_attention(q, *operands[1:]), (operands[0],), (torch.ones_like(operands[0]),))
    assert len(recorder.calls) == 1


@pytest.mark.gpu
def test_forward_mode_is_refused():
    operands = _views(torch.float32, "cuda")["plain"]
    z, index, teacher = torch.randn(2, 3, 9, device="cuda"), torch.zeros(2, 3, 1, dtype=torch.int64, device="cuda"), torch.randn(2, 3, 1, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        for duals in _with_tangents(*operands):
            with pytest.raises(RuntimeError, match="forward-mode"):
                cross_attention(*duals)
        for z_, teacher_ in _with_tangents(z, teacher):
            with pytest.raises(RuntimeError, match="forward-mode"):
                S.distillation_loss_device(z_, index, teacher_)
        assert torch.equal(cross_attention(*operands), cross_attention(*operands))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: S.distillation_loss_device(x, index, teacher), (z,), (torch.ones_like(z),))


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


def half_precision_gradients(q, k, v, dout):
    """Output and gradients of fp16 attention in 64 bits, each with the error that a kernel may have which keeps fp32 sums and rounds to fp16 the output, P, dS
    and the results alone, dS relative to the largest that it is summed with:
      P     half a step, 2^-11; P is formed 2^9 (forward) or 2^14 (backward) times too large, so a subnormal half step is 2^-34 or 2^-39 at most
      dS    half a step, or half a subnormal step, 2^-25, at a scale where the largest of its sum is 2^9 at least: 2^-34 of that one (2^-33 here: the
            largest has its own error)
      rest  fp32: the scores (D + 4 roundings of the sum of absolute values, twice), the exponential (8), the statistic of up to log2 T (2 ln T), dO V and D
            (D roundings; D from the rounded output), the sums over keys or rows (their length)
      results and output: half a step, or half a subnormal step."""
    h, f32, sub = 2.0 ** -11, 2.0 ** -24, 2.0 ** -25
    B, U, H, D = q.shape
    T, Hkv = k.shape[1:3]
    scale, back = D ** -0.5, lambda x: x.permute(0, 2, 1, 3)      # noqa: E731
    wide = lambda x: back(x.double()).repeat_interleave(H // Hkv, 1)      # noqa: E731
    Q, K, V, dO = back(q.double()), wide(k), wide(v), back(dout.double())
    rounded = lambda x: (h * x.abs()).clamp_min(sub) + f32 * x.abs()      # noqa: E731
    P = torch.softmax(scale * Q @ K.transpose(2, 3), -1)
    out = P @ V
    rel = 2 * (D + 4) * f32 * (scale * Q.abs() @ K.abs().transpose(2, 3)).amax(-1, keepdim=True) + 8 * f32
    E_out = rounded(out) + (h + rel + T * f32) * (P @ V.abs()) + 2.0 ** -34 * V.abs().sum(2, keepdim=True)
    dp, delta = dO @ V.transpose(2, 3), (dO * out).sum(-1, keepdim=True)
    ds = P * (dp - delta)
    rel = rel + 2 * math.log(max(T, 2)) * f32
    E_D = (dO.abs() * E_out).sum(-1, keepdim=True) + D * f32 * (dO * out).abs().sum(-1, keepdim=True)
    E = P * (D * f32 * dO.abs() @ V.abs().transpose(2, 3) + E_D) + (rel + 4 * f32) * P * (dp.abs() + delta.abs())
    share = lambda x: x.reshape(B, Hkv, H // Hkv, T, D).sum(2).permute(0, 2, 1, 3)      # noqa: E731
    E_q = E + (h * ds.abs()).maximum(2.0 ** -33 * ds.abs().amax(-1, keepdim=True))
    column = ds.abs().reshape(B, Hkv, -1, T).amax(2)[:, :, None].expand(B, Hkv, H // Hkv, T).reshape(B, H, 1, T)
    E_k = E + (h * ds.abs()).maximum(2.0 ** -33 * column)
    n = U * (H // Hkv) * f32
    dq, dk, dv = scale * ds @ K, share(scale * ds.transpose(2, 3) @ Q), share(P.transpose(2, 3) @ dO)
    return {"out": (back(out), back(E_out)),
            "dq": (back(dq), rounded(back(dq)) + back(scale * (E_q + T * f32 * ds.abs()) @ K.abs())),
            "dk": (dk, rounded(dk) + share(scale * (E_k + n * ds.abs()).transpose(2, 3) @ Q.abs())),
            "dv": (dv, rounded(dv) + share(((h + rel + n) * P + 2.0 ** -39).transpose(2, 3) @ dO.abs()))}


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1.0, 300.0])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 8), (2, 40, 1500, 4, 2, 64), (2, 5, 8000, 4, 2, 64), (1, 600, 600, 2, 1, 32), (2, 200, 300, 2, 1, 128), (3, 37, 129, 8, 2, 96),
                                   (32, 128, 130, 4, 4, 128), (40, 129, 131, 16, 8, 64), (64, 65, 140, 8, 4, 32), (24, 300, 200, 16, 8, 96)], ids=lambda s: "x".join(map(str, s)))
def test_half_precision_gradients_of_any_size(shape, size):
    """Output gradients from a mean over many rows (1e-4) to a scaled loss: entries of dS are far below or above what fp16 holds, their sums are not lost."""
    B, U, T, H, Hkv, D = shape
    g = torch.Generator().manual_seed(34)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    q, k, v, dout = ((r(*s) * f + m).half().cuda() for s, f, m in (((B, U, H, D), 1, 0.3), ((B, T, Hkv, D), 1, 0), ((B, T, Hkv, D), 1, 0), ((B, U, H, D), size, 0)))
    want = half_precision_gradients(q, k, v, dout)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = cross_attention(*leaves)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, dout))):
        value, bound = want[name]
        assert torch.isfinite(got).all(), name
        worst = ((got.double() - value).abs() - bound).max().item()
        assert worst <= 0, f"{name}: {worst:.3g} over the bound"


@pytest.mark.gpu
def test_half_precision_scores_that_grow_along_the_keys():
    """The largest dS of a row, and of a key, comes late: what was summed before at a larger scale is carried over."""
    g = torch.Generator().manual_seed(35)
    B, U, T, H, Hkv, D = 2, 300, 700, 4, 2, 64
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    q, k = r(B, U, H, D), r(B, T, Hkv, D)
    q, k = q * torch.logspace(-2, 0, U)[:, None, None], k * torch.logspace(-3, 0.5, T)[:, None, None]
    v, dout = r(B, T, Hkv, D) * torch.logspace(-3, 1, T)[:, None, None], r(B, U, H, D) * torch.logspace(-4, 1, U)[:, None, None]
    q, k, v, dout = (x.half().cuda() for x in (q, k, v, dout))
    want = half_precision_gradients(q, k, v, dout)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(cross_attention(*leaves), leaves, dout)):
        value, bound = want[name]
        assert ((got.double() - value).abs() <= bound).all(), name


@pytest.mark.gpu
def test_half_precision_terms_beyond_the_type():
    """dS above 65504 whose sums, times small keys and queries and the scale, are far below."""
    g = torch.Generator().manual_seed(36)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    q, k, v = (x.half().cuda() for x in (0.1 * r(2, 3, 2, 64), 0.01 * r(2, 4, 2, 64), 4 * r(2, 4, 2, 64).sign()))
    dout = (3e4 * r(2, 3, 2, 64).sign()).half().cuda()
    want = half_precision_gradients(q, k, v, dout)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(cross_attention(*leaves), leaves, dout)):
        value, bound = want[name]
        assert value.abs().max() < 65504 and torch.isfinite(got).all(), name
        assert ((got.double() - value).abs() <= bound).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(16, 1000, 100, 8, 1, 64), (8, 2100, 200, 8, 1, 32), (5, 4100, 300, 4, 1, 64)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_ranges_of_rows_of_ragged_utterances(dtype, shape):
    """Many rows on few keys of different lengths: ranges of the rows and utterances by length in one launch."""
    q, k, v, dout, lengths = _inputs(dtype, *shape, seed=37)
    _check(q, k, v, dout, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("limits", [dict(top_k=3), dict(top_k=4), dict(top_k=300), dict(top_p=0.9999), dict(top_p=0.5), dict()], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("V", [5, 300, 5000, 20000])
def test_draws_at_distances_beyond_fp32(V, dtype, limits):
    """Logits of both ends of the type at a temperature of its size: 6e38 apart, which fp32 does not hold, and 2^-8.7 of the weight all the same."""
    g = torch.Generator().manual_seed(38)
    z = torch.full((4, V), -math.inf)
    for b in range(4):
        at = torch.randperm(V, generator=g)[:min(V, 400)]
        z[b, at] = (-1.0 + 0.1 * torch.rand(len(at), generator=g)) * 3e38
        z[b, at[0]] = 3e38
    _check_draws(z.to(dtype).cuda(), torch.rand(4, generator=g).cuda(), temperature=1e38, **limits)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [False, True], ids=["one limit", "by row"])
@pytest.mark.parametrize("V", [300, 5000, 20000])
def test_few_candidates_at_distances_beyond_fp32(V, rows):
    """Fewer candidates than top_k may take and all but one of them out of fp32's reach: each random number draws its own."""
    z = torch.full((8, V), -math.inf)
    z[:, 7], z[:, 70], z[:, 200] = 3e38, -3e38, -2.9e38
    # shares of the mass: 1, 2^-8.66 and 2^-8.51 by index
    u = torch.tensor([0.0, 0.5, 0.99, 0.9945, 0.996, 0.9972, 0.9985, 0.9999], device="cuda")
    top_k = torch.full((8,), 3, device="cuda") if rows else 3
    tokens, _ = _check_draws(z.cuda(), u, temperature=1e38, top_k=top_k)
    assert set(tokens.tolist()) == {7, 70, 200}


def test_limits_by_row_of_every_type():
    """What a limit's tensor becomes on its way to the library: int32 or fp32, whatever type it has; other types are refused."""
    cpu = torch.device("cpu")
    for dtype in (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64):
        scalar, address, held = _limit("top_k", torch.tensor([0, 3, 100], dtype=dtype), 3, cpu, whole=True)
        assert scalar == 0 and held.dtype == torch.int32 and held.tolist() == [0, 3, 100] and address == held.data_ptr()
    assert _limit("top_k", torch.tensor([2 ** 40, -2 ** 40, 7]), 3, cpu, whole=True)[2].tolist() == [2 ** 31 - 1, 0, 7]
    assert _limit("top_k", torch.tensor([-128, -1, 7], dtype=torch.int8), 3, cpu, whole=True)[2].tolist() == [0, 0, 7]
    for dtype in (torch.float16, torch.bfloat16, torch.float32, torch.float64):
        assert _limit("top_p", torch.tensor([0.0, 0.5, 1.0], dtype=dtype), 3, cpu)[2].tolist() == [0.0, 0.5, 1.0]
    for dtype in (torch.bool, torch.complex64, torch.float32):
        with pytest.raises(RuntimeError, match="top_k must be"):
            _limit("top_k", torch.ones(3).to(dtype), 3, cpu, whole=True)
    for dtype in (torch.bool, torch.complex64, torch.int64):
        with pytest.raises(RuntimeError, match="top_p must be"):
            _limit("top_p", torch.ones(3).to(dtype), 3, cpu)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16], ids=lambda t: str(t)[6:])
def test_top_k_by_row_of_narrow_types(dtype):
    g = torch.Generator().manual_seed(39)
    z, u = torch.randn(5, 900, generator=g).cuda() * 2, torch.rand(5, generator=g).cuda()
    top_k = torch.tensor([0, 1, 2, 50, 127], device="cuda")
    for a, b in zip(sample_tokens(z, u, top_k=top_k.to(dtype)), sample_tokens(z, u, top_k=top_k)):
        assert torch.equal(a, b)


def test_sizes_that_the_library_would_take_for_smaller_ones():
    """2^32 + 5 would arrive as 5: nothing is planned for it (stride 0: such a tensor costs no memory)."""
    x = torch.zeros(1, 1, 1, 8)
    plan = lambda q, k: ca._plan(q.shape, k.shape, k.shape, q.stride(), k.stride(), k.stride(), q.dtype, None)      # noqa: E731
    assert plan(x, x.expand(1, 5, 1, 8)) is not None
    for n in (2 ** 32 + 5, 2 ** 31, 2 ** 30):
        assert plan(x, x.expand(1, n, 1, 8)) is None and plan(x.expand(1, n, 1, 8), x) is None
        assert plan(x.expand(n, 1, 1, 8), x.expand(n, 1, 1, 8)) is None and plan(x.expand(1, 1, n, 8), x) is None


@pytest.mark.gpu
def test_sizes_beyond_32_bits_are_refused():
    x, z = torch.zeros(1, 1, 1, 8, device="cuda"), torch.zeros(1, 1, device="cuda")
    index = torch.zeros(1, 1, 1, dtype=torch.int64, device="cuda")
    for n in (2 ** 32 + 5, 2 ** 30):
        for q, k in ((x, x.expand(1, n, 1, 8)), (x.expand(1, n, 1, 8), x), (x.expand(n, 1, 1, 8), x.expand(n, 1, 1, 8)), (x.expand(1, 1, n, 8), x)):
            with pytest.raises(RuntimeError, match="2\\^30"):
                cross_attention(q, k, k)
        for shape in ((1, n), (n, 1)):
            with pytest.raises(RuntimeError, match="2\\^30"):
                sample_tokens(z.expand(shape), z[0].expand(shape[0]))
        for shape in ((n, 1, 1), (1, n, 1), (1, 1, n)):
            with pytest.raises(RuntimeError, match="2\\^30"):
                S.distillation_loss_device(z[None].expand(shape), index.expand(*shape[:2], 1), z[None].expand(*shape[:2], 1))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [30, 700, 70000])
@pytest.mark.parametrize("K", [1, 5])
def test_a_teacher_that_is_not_a_number_is_not_silent(V, K):
    """A row whose entries are all NaN teaches NaN, as the formula says, not nothing; absent entries may hold anything."""
    g = torch.Generator().manual_seed(41)
    z, teacher = torch.randn(2, 3, V, generator=g).cuda(), torch.randn(2, 3, K, generator=g).cuda()
    index = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(6)]).view(2, 3, K).cuda()

    def step(teacher, index):
        x = z.clone().requires_grad_(True)
        loss = S.distillation_loss_device(x, index, teacher, 2.0)
        return loss.item(), torch.autograd.grad(loss, (x,))[0]

    want_loss, want = step(teacher, index)
    for entries in (slice(None), slice(0, 1)):
        bad = teacher.clone()
        bad[1, 2, entries] = math.nan
        loss, grad = step(bad, index)
        assert math.isnan(loss)
        taught = torch.zeros_like(z, dtype=torch.bool)
        taught[1, 2, index[1, 2]] = True
        assert torch.equal(grad.isnan(), taught) and torch.equal(grad[~taught], want[~taught])
    absent, none = index.clone(), teacher.clone()
    absent[0, 1], none[0, 1] = -1, math.nan
    kept = teacher.clone()
    kept[0, 1] = 0.0
    assert math.isfinite(step(none, absent)[0]) and step(none, absent)[0] == step(kept, absent)[0]
    assert not step(none, absent)[1][0, 1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("U, T", [(1, 6), (1, 1500), (40, 70), (150, 1500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_keys_whose_scores_are_all_minus_infinity(dtype, U, T):
    """0 / 0: NaN in the output and in the gradients of that utterance; zeros remain those of an utterance without frames; the others keep their bits."""
    q, k, v, dout, _ = _inputs(dtype, 4, U, T, 4, 2, 64, seed=42)
    q = q.abs() + 0.5
    lengths = torch.tensor([T, T // 2, 0, T], dtype=torch.int32, device="cuda")

    def step(k):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = cross_attention(*leaves, lengths)
        with torch.no_grad():
            again = cross_attention(*leaves, lengths)
        assert torch.equal(out.isnan(), again.isnan()) and torch.equal(out[~out.isnan()], again[~again.isnan()])
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    want, bad = step(k), k.clone()
    bad[1, :T // 2] = -math.inf
    got = step(bad)
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        for i in (0, 2, 3):
            assert torch.equal(a[i], b[i]), name
        assert (a[1, :T // 2] if name in ("dk", "dv") else a[1]).isnan().all(), name
        assert name in ("out", "dq") or not a[1, T // 2:].any(), name
    assert not got[0][2].any() and not got[1][2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [30, 3001, 140000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_captured_and_eager_gradients_of_a_scaled_loss_are_one(dtype, V):
    """A seed other than one goes into the gradient before its rounding, in a graph and outside: the same kernel, the same bits."""
    g = torch.Generator().manual_seed(43)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()      # noqa: E731
    z, index, teacher = r(3, 5, V).requires_grad_(True), torch.randint(0, V, (3, 5, 7), generator=g).cuda(), r(3, 5, 7)
    lengths, seed = torch.tensor([5, 0, 3], dtype=torch.int32, device="cuda"), torch.tensor(3.0, device="cuda")

    def step():
        loss = S.distillation_loss_device(z, index, teacher, 2.0, lengths)
        return loss.detach(), *torch.autograd.grad(loss, (z,), seed)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for value in (3.0, 1.0, 1.7e-3, 1024.0):
        seed.fill_(value)
        teacher.add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(step(), held):
            assert torch.equal(a, b), value


@pytest.mark.gpu
def test_a_teacher_of_minus_infinities_teaches_nothing():
    z, index = torch.randn(2, 3, 50, generator=torch.Generator().manual_seed(44)).cuda(), torch.arange(6, device="cuda").view(2, 3, 1).repeat(1, 1, 4)
    teacher = torch.randn(2, 3, 4, generator=torch.Generator().manual_seed(45)).cuda()
    results = []
    for t, i in ((-math.inf, index[0, 1]), (0.0, -1)):
        x, told, named = z.clone().requires_grad_(True), teacher.clone(), index.clone()
        told[0, 1], named[0, 1] = t, i
        loss = S.distillation_loss_device(x, named, told)
        results.append((loss.detach(), *torch.autograd.grad(loss, (x,))))
    for a, b in zip(*results):
        assert torch.equal(a, b) and torch.isfinite(a).all()
