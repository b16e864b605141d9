"""Distillation from a teacher's top logits (``distillation_loss_device``) against the formula in 64 bits.

Tolerances (derived).  x = (z - max z) / tau: one difference and one product, relative 2^-23 of |x| <= span; an exponential adds 2^-23 and an
n-term sum of positive terms n' 2^-24 (n' = the longest chain: V / threads + 10, at most V).  So q and p are off by
r = (2 span + 4 + n') 2^-23 relative; a row's loss by p |log| (r + 2^-22) per entry plus the error of both log-sums (r); the gradient by r (q + p) tau w
before it is rounded to its type (half a step, and half the smallest subnormal)."""
import math

import pytest
import torch

from las_pytorch_amd import _cabi
from las_pytorch_amd.solver import solver as S
from las_pytorch_amd.solver.solver import distillation_loss_device

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(z, index, teacher, tau, lengths, upstream=1.0):
    """(loss, its bound, gradient, its bound) in float64, entry by entry as the definition says (absent entries, classes named twice)."""
    B, U, V = z.shape
    f = 2.0 ** -23
    x = z.double() / tau
    present = (index >= 0) & (index < V)
    safe = torch.where(present, index, 0).long()
    t = torch.where(present, teacher.double() / tau, -math.inf)
    any_entry = present.any(-1) & (t.amax(-1) > -math.inf)
    t = torch.where(any_entry[..., None], t, 0.0)
    logp = torch.log_softmax(t, -1)
    p = torch.where(present & any_entry[..., None], logp.exp(), 0.0)
    logq = torch.log_softmax(x, -1)
    q = logq.exp()
    at = logq.gather(-1, safe)
    kl = torch.where(p > 0, p * (logp - at), 0.0).sum(-1)
    n = lengths.clamp(0, U)
    counts = (torch.arange(U, device=z.device) < n[:, None]) & any_entry
    w = torch.where(counts, 1.0 / (B * n[:, None].clamp_min(1)).double(), 0.0)
    loss = (w * kl).nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf).sum() * tau * tau
    target = torch.zeros_like(x).scatter_add_(-1, safe, p)
    grad = (tau * upstream * w)[..., None] * (q - target)
    finite = lambda v: torch.where(v.isfinite(), v, 0.0)      # noqa: E731
    span = finite((x.amax(-1, keepdim=True) - x)).amax(-1)
    chain = min(V, V // 64 + 10) if V <= 2048 else V // 256 + 10
    r = (2 * span + 4 + chain) * f + (2 * finite(t.amax(-1, keepdim=True) - t).amax(-1) + 4 + index.shape[2]) * f
    bound_loss = (tau * tau * w * ((finite(p * (logp.abs() + at.abs())).sum(-1)) * (r + 2 * f) + 2 * r)).sum() + 4 * f * abs(loss)
    h = torch.finfo(z.dtype).eps / 2
    sub = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps / 2
    bound = (abs(tau * upstream) * w * (r + 4 * f))[..., None] * (q + target) + h * grad.abs() + sub
    return loss, bound_loss, grad, bound


def _case(dtype, B, U, V, K, seed=0, tdtype=None, idx=torch.int64):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(B, U, V, generator=g) * 3).to(dtype).cuda()
    index = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(B * U)]).view(B, U, K).to(idx).cuda()
    teacher = (torch.randn(B, U, K, generator=g) * 2).to(tdtype or dtype).cuda()
    lengths = torch.randint(0, U + 1, (B,), generator=g).to(torch.int32)
    lengths[0] = U
    if B > 1:
        lengths[1] = 0
    return z, index, teacher, lengths.cuda()


def _check(z, index, teacher, tau, lengths, seed=1.0):
    loss_w, bl, grad_w, bg = reference(z, index, teacher, tau, lengths, seed)
    zl = z.detach().requires_grad_(True)
    loss = distillation_loss_device(zl, index, teacher, tau, lengths)
    (grad,) = torch.autograd.grad(loss, (zl,), torch.tensor(seed, device="cuda"))
    assert loss.dtype == torch.float32 and loss.shape == () and grad.dtype == z.dtype and grad.shape == z.shape
    assert abs(loss.double() - loss_w) <= bl, (loss.item(), loss_w.item(), bl.item())
    err = (grad.double() - grad_w).abs()
    assert torch.isfinite(grad).all()
    assert (err <= bg).all(), f"{(err - bg).max().item():.3g} over the bound (largest error {err.max().item():.3g})"
    with torch.no_grad():
        assert torch.equal(distillation_loss_device(z, index, teacher, tau, lengths), loss.detach())
    return loss.detach(), grad


# vocabularies on both sides of every launch size, odd ones among them
SIZES = [(1, 1, 1, 1), (3, 5, 2, 2), (4, 7, 30, 8), (2, 3, 257, 3), (3, 4, 513, 200), (2, 3, 1031, 64), (2, 3, 4097, 33), (2, 2, 8200, 5), (2, 2, 16390, 1024),
         (2, 2, 32771, 16), (2, 2, 65541, 64), (2, 2, 131075, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_loss_and_gradient(dtype, size):
    _check(*_case(dtype, *size)[:3], 2.0, _case(dtype, *size)[3])


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [0.5, 1.0, 4.0])
@pytest.mark.parametrize("tdtype", TYPES, ids=lambda t: str(t)[6:])
def test_types_of_the_teacher_and_temperatures(tdtype, tau):
    z, index, teacher, lengths = _case(torch.bfloat16, 3, 6, 300, 17, seed=1, tdtype=tdtype, idx=torch.int32)
    a, ga = _check(z, index, teacher, tau, lengths)
    b, gb = _check(z, index.long(), teacher, tau, lengths.long())
    assert torch.equal(a, b) and torch.equal(ga, gb)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 700, 5003])
def test_absent_entries_and_classes_named_twice(V):
    z, index, teacher, lengths = _case(torch.float32, 3, 6, V, 12, seed=2)
    index[0, 0, 3:] = -1                      # a short row
    index[0, 1, 0] = V                        # outside the vocabulary
    index[0, 2] = -1                          # no entry at all
    index[0, 3] = 5                           # one class twelve times
    index[0, 4, 6:] = index[0, 4, :6]         # six classes twice
    teacher[0, 5, 2:9] = -math.inf            # entries of no probability
    loss, grad = _check(z, index, teacher, 1.5, lengths)
    assert not grad[0, 2].any() and not grad[1].any()
    far = index.clone()
    far[0, 1, 0] = 2 ** 40
    far[0, 0, 3:] = -2 ** 40
    assert torch.equal(distillation_loss_device(z, far, teacher, 1.5, lengths), loss)


@pytest.mark.gpu
def test_masked_classes():
    """Logits of -inf (a masked vocabulary): no probability, no gradient; a taught class among them makes the loss infinite, not NaN."""
    z, index, teacher, lengths = _case(torch.float32, 2, 3, 600, 4, seed=3)
    lengths[1] = 3
    index[:] = torch.tensor([1, 3, 5, 7], device="cuda")
    z[..., 0::2] = -math.inf
    _, grad = _check(z, index, teacher, 1.0, lengths)
    assert not grad[..., 0::2].any()
    index[0, 0, 0] = 4
    zl = z.requires_grad_(True)
    loss = distillation_loss_device(zl, index, teacher, 1.0, lengths)
    (grad,) = torch.autograd.grad(loss, (zl,))
    assert loss.item() == math.inf and torch.isfinite(grad).all() and grad[0, 0, 4] < 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_views_of_the_decode_kernels_buffer(dtype):
    """(U,B,V) seen as (B,U,V), a slice of a wider buffer at an odd offset, and a vocabulary that is not the last dimension."""
    z, index, teacher, lengths = _case(dtype, 3, 5, 31, 6, seed=4)
    want, gwant = _check(z, index, teacher, 2.0, lengths)
    wide = torch.zeros(3, 5, 40, device="cuda", dtype=dtype)
    wide[..., 3:34] = z
    for view in (z.transpose(0, 1).contiguous().transpose(0, 1), wide[..., 3:34], z.transpose(1, 2).contiguous().transpose(1, 2)):
        v = view.detach().requires_grad_(True)
        loss = distillation_loss_device(v, index, teacher, 2.0, lengths)
        (g,) = torch.autograd.grad(loss, (v,))
        assert torch.equal(loss, want) and torch.equal(g, gwant)
    i2, t2 = index.transpose(0, 1).contiguous().transpose(0, 1), teacher.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(distillation_loss_device(z, i2, t2, 2.0, lengths), want)


@pytest.mark.gpu
def test_seeds_and_retained_graphs():
    z, index, teacher, lengths = _case(torch.float32, 3, 4, 900, 5, seed=5)
    for seed in (1.0, -2.5, 0.0):
        _check(z, index, teacher, 2.0, lengths, seed)
    zl = z.detach().requires_grad_(True)
    loss = distillation_loss_device(zl, index, teacher, 2.0, lengths)
    (first,) = torch.autograd.grad(loss, (zl,), retain_graph=True)
    kept = first.clone()
    (second,) = torch.autograd.grad(2 * loss, (zl,), retain_graph=True)
    (third,) = torch.autograd.grad(loss, (zl,))
    assert torch.equal(first, kept) and torch.equal(third, first) and first.data_ptr() != third.data_ptr()
    err = (second.double() - 2 * first.double()).abs()
    assert (err <= 2.0 ** -21 * first.abs()).all()       # formed again with the factor inside: a few roundings apart
    (g,) = torch.autograd.grad(distillation_loss_device(zl, index, teacher, 2.0, lengths), (zl,), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_scaled_losses(dtype):
    """Seeds of a scaled or weighted loss: the gradient is rounded to its type once, with the seed inside.  (V = 4097: most unscaled entries lie below
    what fp16 can hold; 4 x 7 steps: the largest entry, 65536 / 4, lies within it.)"""
    z, index, teacher, lengths = _case(dtype, 4, 7, 4097, 8, seed=9)
    for seed in (65536.0, -2.5, 1 / 3, 2.0 ** -12):
        _check(z, index, teacher, 1.0, lengths, seed)


@pytest.mark.gpu
def test_gradient_against_differences():
    """Against central differences of the formula in 64 bits, along a random direction (step 1e-5)."""
    z, index, teacher, lengths = _case(torch.float32, 2, 3, 50, 7, seed=6)
    _, grad = _check(z, index, teacher, 2.0, lengths)
    d = torch.randn(z.shape, generator=torch.Generator().manual_seed(7)).cuda().double()
    f = lambda s: reference64(z.double() + s * d, index, teacher, 2.0, lengths)      # noqa: E731
    diff = ((f(1e-5) - f(-1e-5)) / 2e-5).item()
    bound = (reference(z, index, teacher, 2.0, lengths)[3] * d.abs()).sum().item()
    assert abs((grad.double() * d).sum().item() - diff) <= bound + 1e-8 * (1 + abs(diff))


def reference64(z, index, teacher, tau, lengths):
    return reference(z, index, teacher, tau, lengths)[0]


@pytest.mark.gpu
def test_streams_and_graphs():
    z, index, teacher, lengths = _case(torch.bfloat16, 4, 9, 3001, 20, seed=8)
    zl = z.detach().requires_grad_(True)

    def step():
        loss = distillation_loss_device(zl, index, teacher, 2.0, lengths)
        return loss.detach(), *torch.autograd.grad(loss * 3.0, (zl,))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        teacher.add_(torch.linspace(0, 1, 20, device="cuda").to(teacher.dtype))
        graph.replay()
        torch.cuda.synchronize()
        loss, grad = step()
        assert torch.equal(loss, held[0]), i
        # (the graph's backward has the factor inside, the eager one multiplies a gradient that is rounded to bf16 already: a step of 2^-8 apart)
        assert ((grad.float() - held[1].float()).abs() <= 2.0 ** -7 * held[1].float().abs()).all(), i


@pytest.mark.gpu
def test_a_backward_captured_alone():
    """Forward eager, backward in a graph: every replay gives the same gradient (nothing is multiplied twice), and follows its seed.  The forward
    runs on the stream that captures: autograd runs a backward on its forward's stream, and work on any other stream ends a capture."""
    z, index, teacher, lengths = _case(torch.float32, 3, 5, 700, 6, seed=10)
    seed = torch.tensor(2.0, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        zl = z.detach().requires_grad_(True)
        loss = distillation_loss_device(zl, index, teacher, 2.0, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (held,) = torch.autograd.grad(loss, (zl,), seed, retain_graph=True)
    for value in (2.0, 2.0, -3.0):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        _, _, want, bound = reference(z, index, teacher, 2.0, lengths, value)
        assert ((held.double() - want).abs() <= bound).all(), value
    (eager,) = torch.autograd.grad(loss, (zl,), torch.tensor(1.0, device="cuda"))
    torch.cuda.synchronize()
    _, _, want, bound = reference(z, index, teacher, 2.0, lengths)
    assert ((eager.double() - want).abs() <= bound).all()


@pytest.mark.gpu
def test_beside_the_smoothed_loss_of_a_speller_step():
    """The two losses of a taught training step on one (U,B,V) buffer of log-probs: gradients add."""
    U, B, V = 7, 3, 30
    g = torch.Generator().manual_seed(9)
    buf = torch.log_softmax(torch.randn(U, B, V, generator=g), -1).cuda().requires_grad_(True)
    labels = torch.nn.functional.one_hot(torch.randint(2, V, (B, U), generator=g), V).cuda()
    z, index, teacher, lengths = _case(torch.float32, B, U, V, 5, seed=9)
    logp = S.stack_steps(list(buf.unbind(0)), U)
    assert logp.data_ptr() == buf.data_ptr()
    a, b = S.label_smoothing_loss_device(logp, labels, 0.1), distillation_loss_device(logp, index, teacher, 2.0, lengths)
    (ga,) = torch.autograd.grad(a, (buf,), retain_graph=True)
    (gb,) = torch.autograd.grad(b, (buf,), retain_graph=True)
    (gc,) = torch.autograd.grad(a + b, (buf,))
    assert (gc - (ga + gb)).abs().max() <= 2.0 ** -23 * (ga.abs() + gb.abs()).max() * 2
    want = reference(buf.detach().transpose(0, 1), index, teacher, 2.0, lengths)
    assert ((gb.transpose(0, 1).double() - want[2]).abs() <= want[3]).all()


@pytest.mark.gpu
def test_refusals():
    z, index, teacher, lengths = _case(torch.float32, 2, 3, 20, 4)
    good = dict(pred_y=z, teacher_index=index, teacher_logits=teacher, temperature=1.0, lengths=lengths)
    for change, message in [
        (dict(pred_y=z.cpu()), "no CPU fallback"), (dict(pred_y=z[0]), "B,U,V"), (dict(pred_y=z.double()), "fp32, bf16 or fp16"),
        (dict(teacher_index=index[:, :2]), "must"), (dict(teacher_index=index[..., :2]), "must"), (dict(teacher_index=index.short()), "int32 or int64"),
        (dict(teacher_logits=teacher.double()), "int32 or int64"), (dict(teacher_logits=teacher.clone().requires_grad_(True)), "teacher"),
        (dict(temperature=0.0), "positive"), (dict(temperature=-1.0), "positive"), (dict(temperature=math.nan), "positive"), (dict(temperature=math.inf), "positive"),
        (dict(teacher_index=index[..., :0], teacher_logits=teacher[..., :0]), "entries"), (dict(pred_y=z[..., :0]), "row"),
        (dict(teacher_index=index.repeat(1, 1, 257), teacher_logits=teacher.repeat(1, 1, 257)), "entries"),
        (dict(lengths=lengths[:1]), "lengths"), (dict(lengths=lengths.float()), "lengths"), (dict(lengths=lengths.cpu()), "device"),
        (dict(teacher_index=index.cpu()), "device"), (dict(teacher_logits=teacher.cpu()), "device"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            distillation_loss_device(**{**good, **change})


def test_c_entry_refuses_before_it_launches():
    """Status 1 and a message, nothing touched (runs without a GPU)."""
    L = _cabi.lib()
    shape = dict(B=1, U=1, V=8, K=2, dtype=0, teacher_dtype=0, index_64=1, temperature=1.0, stride_b=8, stride_u=8, dstride_b=8, dstride_u=8)
    names = ["logits", "index", "teacher", "lengths", "loss", "dlogits", "upstream", "scratch", "stream"]
    good = dict(logits=4096, index=4096, teacher=4096, lengths=None, loss=4096, dlogits=4096, upstream=4096, scratch=4096, stream=None)
    for change in (dict(dtype=3), dict(dtype=-1), dict(teacher_dtype=3), dict(B=0), dict(U=0), dict(V=0), dict(V=1 << 30), dict(K=0), dict(K=1025),
                   dict(temperature=0.0), dict(temperature=1e-35), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(B=1 << 20, U=1 << 20)):
        d = _cabi.DistillDesc(**{**shape, **change})
        assert L.las_distill_loss(d, *(good[n] for n in names)) == 1, change
        assert L.las_distill_grad_unless_one(d, *(good[n] for n in names if n not in ("loss", "scratch"))) == 1, change
        assert b"distillation" in L.las_last_error()
    d = _cabi.DistillDesc(**shape)
    for change in (dict(logits=None), dict(index=None), dict(teacher=None), dict(loss=None, dlogits=None), dict(scratch=None)):
        assert L.las_distill_loss(d, *({**good, **change}[n] for n in names)) == 1, change
        assert b"distillation" in L.las_last_error()
    for change in (dict(logits=None), dict(index=None), dict(teacher=None), dict(dlogits=None), dict(upstream=None)):
        assert L.las_distill_grad_unless_one(d, *({**good, **change}[n] for n in names if n not in ("loss", "scratch"))) == 1, change
    assert L.las_distill_loss(None, *(good[n] for n in names)) == 1
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        distillation_loss_device(torch.zeros(1, 1, 4), torch.zeros(1, 1, 2, dtype=torch.int64), torch.zeros(1, 1, 2))


def test_reference_against_autograd():
    """The formula this file compares with, against autograd in 64 bits (on the CPU)."""
    g = torch.Generator().manual_seed(0)
    z = torch.randn(2, 3, 9, generator=g, dtype=torch.float64).requires_grad_(True)
    index = torch.stack([torch.randperm(9, generator=g)[:4] for _ in range(6)]).view(2, 3, 4)
    teacher = torch.randn(2, 3, 4, generator=g, dtype=torch.float64)
    lengths = torch.tensor([3, 2])
    loss, _, grad, _ = reference(z.detach(), index, teacher, 2.0, lengths)
    want = 0.0
    for b, n in enumerate(lengths.tolist()):
        p = torch.softmax(teacher[b, :n] / 2, -1)
        logq = torch.log_softmax(z[b, :n] / 2, -1).gather(-1, index[b, :n])
        want = want + 4 * torch.nn.functional.kl_div(logq, p, reduction="sum") / (2 * n)
    assert abs(loss - want) < 1e-13
    assert (torch.autograd.grad(want, z)[0] - grad).abs().max() < 1e-13
