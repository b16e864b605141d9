"""Attention of decoder states over an encoder's states (``cross_attention``) against the formula in 64 bits.

Tolerances (derived, per element).  ``h`` is half a step of the type (0 where nothing is rounded to 16 bits).  With ``P`` the exact
probabilities and absolute values taken inside every sum:
  e    relative error of one probability: the score is a D-term fp32 sum of |q||k| (D + 4 roundings at 2^-24 of the sum of absolute
       values), twice (numerator and normaliser), plus the exponential's argument and value;
  out  h |out| + (h + e + T 2^-24) sum_j P |v|                        (P rounded to the type, T-term sum, output rounded)
  e    in the backward also 2 ln T 2^-24: P = 2^(s - lse), lse is up to log2 T beside the scores, and it and the difference are each rounded at that size
  ds   h |ds| + P (E_dp + E_D) + e P (|dp| + |D|),  E_dp = D 2^-24 |do||v|,  E_D = (h + D 2^-24) sum |do||out|  (D from the rounded out)
  fp16 only: what is rounded to it below 2^-14 is off by up to half a subnormal step, 2^-25 (``sub``): each ds; each P, which the kernels form
       too large, by 2^9 in the forward, 2^14 in the backward: by 2^-34 of the row's largest (P is taken relative to a maximum of the row's scores), 2^-39
  dq, dk, dv: the type's half step of the result plus those errors times the other factor, plus the sum's own length times 2^-24."""
import math

import pytest
import torch

import las_pytorch_amd
from las_pytorch_amd import _cabi, cross_attention

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _half(dtype):
    return torch.finfo(dtype).eps / 2 if dtype in (torch.bfloat16, torch.float16) else 0.0


def reference(q, k, v, lengths, dout=None, scale=None):
    """Values and error bounds in float64: {"out": (value, bound), "dq": ..., "dk": ..., "dv": ...}."""
    h, f32 = _half(q.dtype), 2.0 ** -24
    sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    B, U, H, D = q.shape
    T, Hkv = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    keep = (torch.arange(T, device=q.device) < lengths[:, None])[:, None, None, :]
    clean = lambda x: torch.where(keep.reshape(B, T, 1, 1), x.double(), 0.0).permute(0, 2, 1, 3).repeat_interleave(H // Hkv, 1)      # noqa: E731
    Q, K, V = q.double().permute(0, 2, 1, 3), clean(k), clean(v)                       # (B,H,U,D), (B,H,T,D)
    s = torch.where(keep, scale * Q @ K.transpose(2, 3), -math.inf)
    m = s.amax(-1, keepdim=True) if T else torch.zeros(B, H, U, 1, device=q.device, dtype=torch.float64)
    e = torch.where(keep, (s - torch.where(m.isinf(), 0.0, m)).exp(), 0.0)
    P = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    out = P @ V
    absP = scale * Q.abs() @ K.abs().transpose(2, 3)
    rel = (2 * ((D + 4) * f32 * absP.amax(-1, keepdim=True) if T else 0.0) + 8 * f32)
    E_out = (h + f32) * out.abs() + (h + rel + T * f32) * (P @ V.abs()) + sub * 2.0 ** -9 * V.abs().sum(2, keepdim=True)
    back = lambda x: x.permute(0, 2, 1, 3)      # noqa: E731
    res = {"out": (back(out), back(E_out))}
    if dout is None:
        return res
    dO = dout.double().permute(0, 2, 1, 3)
    dp = dO @ V.transpose(2, 3)
    delta = (dO * out).sum(-1, keepdim=True)
    ds = P * (dp - delta)
    E_dp = D * f32 * dO.abs() @ V.abs().transpose(2, 3)
    E_D = (dO.abs() * E_out).sum(-1, keepdim=True) + D * f32 * (dO.abs() * out.abs()).sum(-1, keepdim=True)
    rel = rel + 2 * math.log(max(T, 2)) * f32
    E_ds = h * ds.abs() + P * (E_dp + E_D) + (rel + 4 * f32) * P * (dp.abs() + delta.abs()) + sub * keep
    E_p = (h + rel) * P + sub * 2.0 ** -14 * keep
    share = lambda x: x.reshape(B, Hkv, H // Hkv, T, D).sum(2).permute(0, 2, 1, 3)      # noqa: E731
    n = U * (H // Hkv) * f32
    dq, dk, dv = scale * ds @ K, share(scale * ds.transpose(2, 3) @ Q), share(P.transpose(2, 3) @ dO)
    res["dq"] = back(dq), back((h + f32) * dq.abs() + scale * (E_ds + T * f32 * ds.abs()) @ K.abs())
    res["dk"] = dk, (h + f32) * dk.abs() + share(scale * (E_ds + n * ds.abs()).transpose(2, 3) @ Q.abs())
    res["dv"] = dv, (h + f32) * dv.abs() + share((E_p + n * P).transpose(2, 3) @ dO.abs())
    return res


def _close(got, want, name, tiny):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    err = (got.double() - value).abs()
    worst = (err - bound - tiny).max().item() if err.numel() else -1.0
    assert torch.isfinite(got).all(), name
    assert worst <= 0, f"{name}: {worst:.3g} over the bound (largest error {err.max().item():.3g}, largest bound {bound.max().item():.3g})"


def _tiny(dtype):
    return 0.0 if dtype != torch.float16 else 2.0 ** -24      # fp16 results below its normal range: a step of 2^-24


def _inputs(dtype, B, U, T, H, Hkv, D, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)      # noqa: E731
    lengths = torch.randint(0, T + 1, (B,), generator=g)
    lengths[0] = T
    if B > 1:
        lengths[1] = min(1, T)
    if B > 2:
        lengths[2] = 0
    return r(B, U, H, D), r(B, T, Hkv, D), r(B, T, Hkv, D), r(B, U, H, D), lengths.to(torch.int32).to(device)


def _check(q, k, v, dout, lengths, want=None, scale=None):
    want = want or reference(q, k, v, lengths, dout, scale)
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = cross_attention(q, k, v, lengths, scale)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    tiny = _tiny(q.dtype)
    _close(out.detach(), want["out"], "out", tiny)
    for name, g in zip(("dq", "dk", "dv"), grads):
        _close(g, want[name], name, tiny)
    with torch.no_grad():       # the form without a backward gives the same bits
        assert torch.equal(cross_attention(q, k, v, lengths, scale), out)
    return out, grads


SHAPES = [  # B, U, T, H, Hkv, D
    (1, 1, 1, 1, 1, 8),
    (3, 1, 7, 4, 1, 32),
    (3, 5, 33, 4, 2, 40),
    (4, 130, 65, 2, 2, 64),
    (3, 37, 129, 8, 2, 96),
    (2, 200, 300, 2, 1, 128),
    (3, 3, 257, 6, 2, 104),
    (32, 128, 100, 4, 4, 128),     # enough workgroups for the 128-row / 128-key forms
    (40, 129, 131, 16, 8, 64),
    (64, 65, 140, 8, 4, 32),
    (24, 300, 200, 16, 8, 96),
    (3, 1, 1500, 8, 8, 64),        # split over key ranges
    (3, 2, 2100, 8, 2, 128),
    (3, 1, 1031, 4, 4, 24),
    (32, 70, 200, 8, 8, 128),      # wide heads in the 128-row / 128-key forms
    (2, 150, 1500, 4, 2, 64),      # 128 rows and key ranges
    (1, 100, 1100, 2, 2, 128),
    (2, 9, 300, 4, 4, 96),         # key ranges of fp32 alone
    (2, 700, 40, 4, 2, 64),        # row ranges in the backward
    (1, 1100, 70, 6, 2, 128),
    (3, 4, 1103, 4, 2, 128),       # key ranges in the backward
    (1, 600, 600, 2, 1, 32),       # both
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_values_and_gradients(dtype, shape):
    q, k, v, dout, lengths = _inputs(dtype, *shape)
    _check(q, k, v, dout, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(16, 300, 300, 12, 4, 64), (2, 23, 90, 10, 2, 48), (4, 61, 200, 7, 1, 128), (70, 33, 129, 6, 2, 32)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_groups_that_do_not_divide_a_tile(dtype, shape):
    """Three, five and seven query heads to a key head, rows that span tiles and heads; more utterances than a wave has lanes."""
    q, k, v, dout, lengths = _inputs(dtype, *shape, seed=20)
    _check(q, k, v, dout, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-3, 0.7, 3.0])
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_scales_and_large_scores(dtype, scale):
    """Scales other than the default: nearly flat rows, and rows whose scores grow from tile to tile by far more than the running maximum may lag."""
    q, k, v, dout, lengths = _inputs(dtype, 3, 40, 300, 4, 2, 64, seed=21)
    k = k * torch.linspace(0.1, 1.0, 300, device="cuda").to(dtype)[None, :, None, None]
    _check(q, k, v, dout, lengths, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_what_masked_frames_hold_never_matters(dtype):
    q, k, v, dout, lengths = _inputs(dtype, 5, 9, 70, 4, 2, 64, seed=1)
    lengths = torch.tensor([70, 33, 0, 1, 64], dtype=torch.int32, device="cuda")
    want = reference(q, k, v, lengths, dout)
    lowest = torch.finfo(dtype).min
    for bad in (math.nan, math.inf, -math.inf, lowest):
        kb, vb = k.clone(), v.clone()
        for b, n in enumerate(lengths.tolist()):
            kb[b, n:], vb[b, n:] = bad, bad
        out, (dq, dk, dv) = _check(q, kb, vb, dout, lengths, want)
        for b, n in enumerate(lengths.tolist()):
            assert not dk[b, n:].any() and not dv[b, n:].any()
        assert not out[2].any() and not dq[2].any()


@pytest.mark.gpu
def test_lengths_outside_the_range_and_of_both_types():
    q, k, v, dout, _ = _inputs(torch.float32, 3, 4, 20, 2, 2, 32, seed=2)
    want = cross_attention(q, k, v, torch.tensor([20, 0, 5], dtype=torch.int32, device="cuda"))
    for t, values in ((torch.int32, [100, -3, 5]), (torch.int64, [2 ** 40, -2 ** 40, 5])):
        assert torch.equal(cross_attention(q, k, v, torch.tensor(values, dtype=t, device="cuda")), want)
    assert torch.equal(cross_attention(q, k, v), cross_attention(q, k, v, torch.full((3,), 20, device="cuda")))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_strides_and_alignment(dtype):
    B, U, T, H, Hkv, D = 3, 21, 45, 4, 2, 64
    q, k, v, dout, lengths = _inputs(dtype, B, U, T, H, Hkv, D, seed=3)
    want, grads = _check(q, k, v, dout, lengths)
    fused = torch.stack((k, v), 2)                                            # (B,T,2,Hkv,D): one projection for keys and values
    views = {
        "fused": (q.transpose(1, 2).contiguous().transpose(1, 2), fused[:, :, 0], fused[:, :, 1]),
        "time first": (q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1), v),
        "unaligned": tuple(torch.nn.functional.pad(x, (1, 2))[..., 1:-2] for x in (q, k, v)),
        "columns": tuple(x.transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)),
    }
    for name, (a, b, c) in views.items():
        a, b, c = (x.detach().requires_grad_(True) for x in (a, b, c))
        out = cross_attention(a, b, c, lengths)
        assert torch.equal(out, want), name
        for x, y in zip(torch.autograd.grad(out, (a, b, c), dout.transpose(1, 2).contiguous().transpose(1, 2)), grads):
            assert torch.equal(x, y), name


@pytest.mark.gpu
def test_gradient_against_differences():
    """The derivative along a random direction against central differences of the formula in 64 bits (step 1e-5: their own error is
    below 1e-8 of the scale); the gradient's error is bounded by its elements' bounds times the direction."""
    q, k, v, dout, lengths = _inputs(torch.float32, 3, 6, 40, 4, 2, 32, seed=4)
    want = reference(q, k, v, lengths, dout)
    g = torch.Generator().manual_seed(5)
    d = [torch.randn(x.shape, generator=g).cuda() for x in (q, k, v)]
    xs = [x.detach().requires_grad_(True) for x in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*xs, lengths), xs, dout)
    got = sum((a.double() * b.double()).sum() for a, b in zip(grads, d)).item()
    f = lambda t: (reference(*(x.double() + t * y.double() for x, y in zip((q, k, v), d)), lengths)["out"][0] * dout.double()).sum().item()      # noqa: E731
    diff = (f(1e-5) - f(-1e-5)) / 2e-5
    bound = sum((want[n][1] * b.double().abs()).sum().item() for n, b in zip(("dq", "dk", "dv"), d))
    assert abs(got - diff) <= bound + 1e-7 * abs(diff) + 1e-6


@pytest.mark.gpu
def test_shared_encoder_states_sum_their_gradients():
    """One utterance's states expanded over several hypotheses (stride 0): gradients of the shared tensor are the sum."""
    q, _, _, dout, _ = _inputs(torch.float32, 4, 3, 50, 4, 4, 32, seed=6)
    _, k, v, _, _ = _inputs(torch.float32, 1, 3, 50, 4, 4, 32, seed=7)
    lengths = torch.tensor([50, 20, 1, 0], dtype=torch.int32, device="cuda")
    want = reference(q, k.expand(4, -1, -1, -1), v.expand(4, -1, -1, -1), lengths, dout)
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    out = cross_attention(q, k.expand(4, -1, -1, -1), v.expand(4, -1, -1, -1), lengths)
    _, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    for got, (value, bound) in ((dk, want["dk"]), (dv, want["dv"])):
        value, bound = value.sum(0, keepdim=True), bound.sum(0, keepdim=True)
        _close(got, (value, bound + 4 * 2.0 ** -24 * value.abs() + 1e-9), "shared", 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 20, 90, 4, 2, 64), (40, 129, 131, 16, 8, 64)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_gradients_of_one_side(dtype, shape):
    """A Listener that is not trained (dq alone), frozen decoder states (dk, dv alone): the bits of the full backward."""
    q, k, v, dout, lengths = _inputs(dtype, *shape, seed=8)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    every = torch.autograd.grad(cross_attention(*leaves, lengths), leaves, dout)
    for wanted in ((0,), (1, 2), (2,)):
        xs = [x.detach().requires_grad_(i in wanted) for i, x in enumerate((q, k, v))]
        got = torch.autograd.grad(cross_attention(*xs, lengths), [xs[i] for i in wanted], dout)
        assert all(torch.equal(g, every[i]) for g, i in zip(got, wanted))


@pytest.mark.gpu
def test_empty_sizes():
    for B, U, T in ((0, 3, 5), (2, 0, 5), (2, 3, 0)):
        q, k, v = (torch.randn(B, n, 2, 32, device="cuda", requires_grad=True) for n in (U, T, T))
        out = cross_attention(q, k, v)
        grads = torch.autograd.grad(out.sum(), (q, k, v))
        assert out.shape == q.shape and not out.any() and not any(g.any() for g in grads)
        (dk,) = torch.autograd.grad(cross_attention(q.detach(), k, v.detach()).sum(), (k,))
        assert dk.shape == k.shape and not dk.any()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Frames whose element offset passes 2^31: a view of a large buffer whose utterance stride is 2^31 + 64 elements."""
    stride = 2 ** 31 + 64
    T, Hkv, D = 40, 2, 64
    buf = torch.empty(stride + T * Hkv * D, device="cuda", dtype=torch.bfloat16)
    k = buf.as_strided((2, T, Hkv, D), (stride, Hkv * D, D, 1))
    q, kk, v, dout, _ = _inputs(torch.bfloat16, 2, 3, T, 4, Hkv, D, seed=8)
    k.copy_(kk)
    lengths = torch.tensor([T, 17], dtype=torch.int32, device="cuda")
    assert torch.equal(cross_attention(q, k, v, lengths), cross_attention(q, kk, v, lengths))


@pytest.mark.gpu
def test_streams_graphs_and_repeats():
    """The same bits on another stream, in a replayed graph (forward, one token split over key ranges, backward), and run to run."""
    q, k, v, dout, lengths = _inputs(torch.bfloat16, 3, 40, 150, 4, 2, 64, seed=9)
    q1, k1, v1, _, l1 = _inputs(torch.bfloat16, 3, 1, 1500, 8, 2, 64, seed=10)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]

    def step():
        out = cross_attention(*leaves, lengths)
        return (cross_attention(q1, k1, v1, l1), out.detach(), *torch.autograd.grad(out, leaves, dout))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    for i in range(3):
        q1.add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        again = step()
        for a, b in zip(again, held):
            assert torch.equal(a, b), i


@pytest.mark.gpu
def test_refusals():
    q, k, v, _, lengths = _inputs(torch.float32, 2, 3, 5, 4, 2, 32)
    bad = [
        (dict(query=q.cpu()), "no CPU fallback"),
        (dict(query=q[0]), "must be"),
        (dict(key=k.half()), "share one type"),
        (dict(query=q.double(), key=k.double(), value=v.double()), "fp32, bf16 or fp16"),
        (dict(key=k[:, :4]), "do not go together"),
        (dict(key=k[:1], value=v[:1]), "do not go together"),
        (dict(query=q[:, :, :3]), "do not share"),
        (dict(query=q[..., :30], key=k[..., :30], value=v[..., :30]), "head size"),
        (dict(query=torch.zeros(2, 3, 4, 132, device="cuda"), key=torch.zeros(2, 5, 2, 132, device="cuda"), value=torch.zeros(2, 5, 2, 132, device="cuda")),
         "head size"),
        (dict(scale=0.0), "scale"), (dict(scale=-0.5), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
        (dict(key_lengths=lengths.float()), "key_lengths"),
        (dict(key_lengths=lengths[:1]), "key_lengths"),
        (dict(key_lengths=lengths.cpu()), "key_lengths"),
    ]
    for change, message in bad:
        with pytest.raises(RuntimeError, match=message):
            cross_attention(**{**dict(query=q, key=k, value=v, key_lengths=lengths), **change})
    x = q.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(cross_attention(x, k, v).sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                       # once differentiable


def test_c_entry_refuses_before_it_launches():
    """Argument checks of the C entry points: status 1 and a message, nothing touched (runs without a GPU)."""
    L = _cabi.lib()
    good = dict(B=1, U=1, T=1, H=2, Hkv=1, D=32, dtype=0, scale=1.0, q_b=64, q_u=64, q_h=32, k_b=32, k_t=32, k_h=32, v_b=32, v_t=32, v_h=32)
    for change in (dict(dtype=3), dict(H=3, Hkv=2), dict(Hkv=0), dict(D=0), dict(D=132), dict(D=30), dict(dtype=1, D=20), dict(B=-1), dict(q_u=65),
                   dict(U=1 << 30), dict(T=1 << 30), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)):
        d = _cabi.CrossAttentionDesc(**{**good, **change})
        assert L.las_cross_attention_fwd(d, 4096, 4096, 4096, None, 4096, None, None, None) == 1, change
        assert L.las_cross_attention_bwd(d, 4096, 4096, 4096, None, 4096, 4096, 4096, 4096, 4096, 4096, 4096, None) == 1, change
        assert b"cross attention" in L.las_last_error()
    d = _cabi.CrossAttentionDesc(**good)
    for at in range(3):
        ptrs = [4096] * 3
        ptrs[at] = None
        assert L.las_cross_attention_fwd(d, *ptrs, None, 4096, None, None, None) == 1
        ptrs[at] = 4100
        assert L.las_cross_attention_fwd(d, *ptrs, None, 4096, None, None, None) == 1
    assert L.las_cross_attention_fwd(d, 4096, 4096, 4096, None, None, None, None, None) == 1
    assert L.las_cross_attention_bwd(d, 4096, 4096, 4096, None, 4096, None, 4096, 4096, 4096, 4096, None, None) == 1
    for grads in ((None, 4096, None), (4096, None, 4096), (None, None, None)):       # half of a side, nothing at all
        assert L.las_cross_attention_bwd(d, 4096, 4096, 4096, None, 4096, 4096, 4096, *grads, None, None) == 1
    assert L.las_cross_attention_fwd(None, 4096, 4096, 4096, None, 4096, None, None, None) == 1
    assert L.las_cross_attention_workspace_floats(d) == 0
    assert L.las_cross_attention_workspace_floats(_cabi.CrossAttentionDesc(**{**good, "T": 4096})) > 0
    assert L.las_cross_attention_bwd_workspace_floats(d) == 0
    for long in (dict(T=4096), dict(U=4096)):        # a few rows over many keys, many rows over a few keys: partial sums want a workspace
        d = _cabi.CrossAttentionDesc(**{**good, **long})
        assert L.las_cross_attention_bwd_workspace_floats(d) > 0
        for workspace in (None, 4100):
            assert L.las_cross_attention_bwd(d, 4096, 4096, 4096, None, 4096, 4096, 4096, 4096, 4096, 4096, workspace, None) == 1
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cross_attention(*(torch.zeros(1, 2, 2, 32) for _ in range(3)))
    assert "cross_attention" in las_pytorch_amd.__all__


def test_reference_against_autograd():
    """The formula this file compares with, against autograd of a plain softmax in 64 bits (on the CPU)."""
    q, k, v, dout, _ = _inputs(torch.float64, 2, 4, 9, 4, 2, 8, device="cpu")
    lengths = torch.tensor([9, 4], dtype=torch.int32)
    want = reference(q, k, v, lengths, dout)
    xs = [x.requires_grad_(True) for x in (q, k, v)]
    outs = []
    for b, n in enumerate(lengths.tolist()):
        kb, vb = (x[b, :n].repeat_interleave(2, 1) for x in xs[1:])
        outs.append(torch.einsum("hut,thd->uhd", torch.softmax(torch.einsum("uhd,thd->hut", xs[0][b], kb) / math.sqrt(8), -1), vb))
    out = torch.stack(outs)
    for got, name in zip((out, *torch.autograd.grad(out, xs, dout)), ("out", "dq", "dk", "dv")):
        assert (got - want[name][0]).abs().max() < 1e-12, name
