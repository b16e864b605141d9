"""The decoder operators together, as a program would use them: a student decoder attends over a Listener's features, is taught by a larger model's
top logits beside the smoothed labels, and then draws sequences one token at a time."""
import math

import pytest
import torch

from hip_util import build_las
from las_pytorch_amd import cross_attention, sample_tokens, synth
from las_pytorch_amd.solver import solver as S


def _weights(E, H, Hkv, D, V, dtype, device="cuda"):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[0])).to(dtype).to(device)      # noqa: E731
    return dict(embed=r(V, E), wq=r(E, H * D), wk=r(E, Hkv * D), wv=r(E, Hkv * D), wo=r(H * D, V))


def _student(feat, tokens, lengths, w, H, Hkv, D, attend):
    """Logits (B,U,V) of a one-layer decoder: embedded tokens attend over the features."""
    B, U = tokens.shape
    q = (w["embed"][tokens] @ w["wq"]).view(B, U, H, D)
    k, v = ((feat @ w[n]).view(B, -1, Hkv, D) for n in ("wk", "wv"))
    return attend(q, k, v, lengths).reshape(B, U, H * D) @ w["wo"]


def _plain_attend(q, k, v, lengths):
    share = q.shape[2] // k.shape[2]
    k, v = (x.repeat_interleave(share, 2).permute(0, 2, 1, 3) for x in (k, v))
    s = q.permute(0, 2, 1, 3) @ k.transpose(2, 3) / math.sqrt(q.shape[-1])
    keep = (torch.arange(k.shape[2], device=k.device) < lengths[:, None])[:, None, None]
    p = torch.softmax(torch.where(keep, s, -1e300), -1) * keep
    return (p @ v).permute(0, 2, 1, 3)


@pytest.mark.gpu
def test_taught_step_and_drawing():
    B, U, H, Hkv, D = 3, 7, 4, 2, 16
    c = synth.CONFIGS["tiny"]
    las = build_las(c, synth.make_state_dict(synth.config_shapes("tiny"), seed=17), max_label_len=U)
    x = torch.from_numpy(synth.make_inputs(B, 64, c["F"], seed=17)).cuda()
    feat = las.listener(x)
    V, E = c["V"], feat.shape[2]
    idx, lens = synth.make_labels(B, U, V, seed=5, ragged=True)
    onehot = torch.from_numpy(synth.onehot_labels(idx, lens, V)).cuda()
    labels, steps = torch.from_numpy(idx).long().cuda(), torch.as_tensor(lens).to(torch.int32).cuda()
    frames = torch.tensor([feat.shape[1], 5, 9], dtype=torch.int32, device="cuda")
    teacher = torch.randn(B, U, V, generator=torch.Generator().manual_seed(1)).cuda() * 2
    top, top_index = teacher.topk(8, -1)
    w = {k: v.requires_grad_(True) for k, v in _weights(E, H, Hkv, D, V, torch.float32).items()}

    # one training step: both losses, gradients of the weights and of the Listener's features
    leaf = feat.detach().requires_grad_(True)
    logits = _student(leaf, labels, frames, w, H, Hkv, D, cross_attention)
    loss = S.distillation_loss_device(logits, top_index, top, 2.0, steps) + S.label_smoothing_loss_device(torch.log_softmax(logits, -1), onehot, 0.1)
    grads = torch.autograd.grad(loss, [leaf, *w.values()])

    leaf64 = feat.detach().double().requires_grad_(True)
    w64 = {k: v.detach().double().requires_grad_(True) for k, v in w.items()}
    logits64 = _student(leaf64, labels, frames, w64, H, Hkv, D, _plain_attend)
    p = torch.softmax(top.double() / 2, -1)
    logq = torch.log_softmax(logits64 / 2, -1).gather(-1, top_index)
    counts = (torch.arange(U, device="cuda") < steps[:, None]) / steps[:, None].clamp_min(1).double() / B
    loss64 = 4 * (counts * (p * (p.log() - logq)).sum(-1)).sum() + S.label_smoothing_loss(torch.log_softmax(logits64, -1), onehot.double(), 0.1)
    want = torch.autograd.grad(loss64, [leaf64, *w64.values()])
    assert abs(loss.item() - loss64.item()) <= 1e-5 * abs(loss64.item())
    # fp32 products of up to E H D = 4096 terms on both sides of the operators: 4096 2^-24 of the largest gradient bounds any one of their sums
    for name, a, b in zip(["feat", *w], grads, want):
        assert (a.double() - b).abs().max() <= 4096 * 2.0 ** -24 * b.abs().max(), name

    # and on through the Listener itself
    loss = S.distillation_loss_device(_student(feat, labels, frames, w, H, Hkv, D, cross_attention), top_index, top, 2.0, steps)
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in las.listener.parameters())

    # drawing, one token at a time: single-row attention and a draw per step, against the whole prefix at once
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        tokens = torch.zeros(B, 1, dtype=torch.int64, device="cuda")
        for _ in range(U):
            u = torch.rand(B, generator=g).cuda()
            step = _student(feat, tokens[:, -1:], frames, w, H, Hkv, D, cross_attention)[:, 0]
            whole = _student(feat, tokens, frames, w, H, Hkv, D, cross_attention)[:, -1]
            assert (step - whole).abs().max() <= 4096 * 2.0 ** -24 * whole.abs().max()
            token, logprob = sample_tokens(step, u, temperature=0.9, top_k=12, top_p=0.95, min_p=0.01)
            full = torch.log_softmax(step / 0.9, -1).gather(-1, token[:, None])[:, 0]
            assert ((0 <= token) & (token < V)).all() and (logprob >= full - 1e-5).all() and (logprob <= 0).all()
            tokens = torch.cat([tokens, token[:, None]], 1)


@pytest.mark.gpu
def test_two_streams_and_one_graph_of_all():
    """Calls of all three on two streams at once, and captured together: the results are those of the calls alone."""
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g).cuda()      # noqa: E731
    q, k, v = r(2, 1, 8, 64).half(), r(2, 2000, 2, 64).half(), r(2, 2000, 2, 64).half()
    z, u = r(3, 50000), torch.rand(3, generator=g).cuda()
    s, index, teacher = r(2, 5, 4000), torch.randint(0, 4000, (2, 5, 9), generator=g).cuda(), r(2, 5, 9)

    def all_three():
        return (cross_attention(q, k, v), *sample_tokens(z, u, 0.8, 0, 0.9), *sample_tokens(z, u, 0.8, 40), S.distillation_loss_device(s, index, teacher, 2.0))

    want = all_three()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(all_three())
    torch.cuda.synchronize()
    for out in got:
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    held = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(all_three())
    for i in range(4):
        u.copy_(torch.rand(3, generator=g))
        for n, graph in enumerate(graphs):
            with torch.cuda.stream(streams[n]):
                streams[n].wait_stream(torch.cuda.current_stream(0))
                graph.replay()
        torch.cuda.synchronize()
        want = all_three()
        for out in held:
            for a, b in zip(out, want):
                assert torch.equal(a, b), i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_saved_tensors_kept_elsewhere(dtype):
    """Saved tensors that come back at another address (kept on the host) and forwards that are run again: the bits of the plain backward."""
    from torch.utils.checkpoint import checkpoint

    g = torch.Generator().manual_seed(12)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()      # noqa: E731
    q, k, v, dout = r(3, 20, 4, 64), r(3, 200, 2, 64), r(3, 200, 2, 64), r(3, 20, 4, 64)
    frames = torch.tensor([200, 0, 77], device="cuda")
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    want = torch.autograd.grad(cross_attention(*leaves, frames), leaves, dout)
    with torch.autograd.graph.save_on_cpu():
        out = cross_attention(*leaves, frames)
    again = checkpoint(lambda *x: cross_attention(*x, frames), *leaves, use_reentrant=False)
    for o in (out, again):
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o, leaves, dout), want))

    index, teacher, steps = torch.randint(0, 700, (3, 5, 6), generator=g).cuda(), r(3, 5, 6), torch.tensor([5, 0, 3], device="cuda")
    for z in (r(3, 5, 700), r(5, 3, 700).transpose(0, 1)):
        z = z.detach().requires_grad_(True)
        (want,) = torch.autograd.grad(S.distillation_loss_device(z, index, teacher, 2.0, steps), (z,))
        with torch.autograd.graph.save_on_cpu():
            loss = S.distillation_loss_device(z, index, teacher, 2.0, steps)
        for keep in (True, False):
            (got,) = torch.autograd.grad(loss, (z,), retain_graph=keep)
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_one_tensor_in_several_places():
    """Keys that are the values and the queries too, and a student whose rows are one: gradients of the shared tensor are the sums."""
    g = torch.Generator().manual_seed(13)
    x, dout = torch.randn(2, 40, 4, 64, generator=g).cuda(), torch.randn(2, 40, 4, 64, generator=g).cuda()
    apart = [x.clone().requires_grad_(True) for _ in range(3)]
    want = torch.autograd.grad(cross_attention(*apart), apart, dout)
    x.requires_grad_(True)
    out = cross_attention(x, x, x)
    (got,) = torch.autograd.grad(out, (x,), dout)
    assert torch.equal(out, cross_attention(*apart))
    assert ((got - sum(want)).abs() <= 2 * 2.0 ** -24 * sum(w.abs() for w in want)).all()       # (two additions, in any order)

    row = torch.randn(1, 1, 300, generator=g).cuda().requires_grad_(True)
    index, teacher = torch.randint(0, 300, (3, 4, 5), generator=g).cuda(), torch.randn(3, 4, 5, generator=g).cuda()
    apart = row.detach().expand(3, 4, 300).contiguous().requires_grad_(True)
    (want,) = torch.autograd.grad(S.distillation_loss_device(apart, index, teacher), (apart,))
    (got,) = torch.autograd.grad(S.distillation_loss_device(row.expand(3, 4, 300), index, teacher), (row,))
    assert ((got - want.sum((0, 1), keepdim=True)).abs() <= 24 * 2.0 ** -24 * want.abs().sum((0, 1), keepdim=True)).all()     # (twelve terms, both ways)
