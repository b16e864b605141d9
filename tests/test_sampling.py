"""Drawing tokens (``sample_tokens``) against the definition, row by row in 64 bits.  Tokens have to be equal: the inputs are drawn so that a
border is nowhere nearer than the kernel's weights resolve (2^-44 of the largest), which ``reference`` asserts.  The log-probability is a quotient of
exact sums, a logarithm and one rounding to fp32: half a step of its value, and 2^-40 for the weights' own resolution."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from hip_util import build_las
from las_pytorch_amd import _cabi, sample_tokens, synth

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference_row(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability, distance of the nearest border relative to the mass it divides)."""
    z = np.where(np.isnan(z), -np.inf, np.asarray(z, np.float64))
    live = np.flatnonzero(z > -np.inf)
    if live.size == 0:
        return -1, -math.inf, 1.0
    order = live[np.argsort(-z[live], kind="stable")]
    if not temperature > 0 or top_k == 1:
        return int(order[0]), 0.0, 1.0
    top = z[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(z[order] == top, 1.0, np.exp((z[order] - top) / temperature))
    near = 1.0
    W = np.array([int(x) for x in np.ldexp(w, 80)], dtype=object)      # whole multiples of 2^-80: sums and borders are exact
    if top_k > 1:
        order, w, W = order[:top_k], w[:top_k], W[:top_k]
    if top_p < 1:
        before, total = W.cumsum() - W, W.sum()
        num, den = float(Fraction(float(top_p)) * total).as_integer_ratio()            # (the share is a product in fp64: 0.9 of 30 is 27)
        near = min([near] + [g for g in np.abs((before * den - num).astype(np.float64)) / float(den * total) if g > 0])      # (met exactly: by both sides)
        keep = np.array(before * den < num, dtype=bool)
        keep[0] = True
        order, w, W = order[keep], w[keep], W[keep]
    if min_p > 0:
        keep = w >= min(min_p, 1.0)
        near = min([near] + [g for g in np.abs(w - min_p) if g > 0])
        order, w, W = order[keep], w[keep], W[keep]
    by_index = np.argsort(order)
    order, W = order[by_index], W[by_index]
    cum = W.cumsum()
    total = cum[-1]
    num, den = (min(max(float(u), 0.0), 1.0) if u == u else 0.0).as_integer_ratio()
    near = min([near] + [g for g in np.abs((cum * den - num * total).astype(np.float64)) / float(den * total) if g > 0 and 0 < num < den])
    over = np.flatnonzero(cum * den > num * total)
    at = int(over[0]) if over.size else len(order) - 1
    while W[at] == 0:
        at -= 1
    return int(order[at]), math.log(int(W[at])) - math.log(int(total)), near


def _check(z, u, clear=1e-12, **limits):
    per_row = lambda v, b: v[b].item() if torch.is_tensor(v) else v      # noqa: E731
    tokens, logp = sample_tokens(z, u, **limits)
    assert tokens.dtype == torch.int64 and logp.dtype == torch.float32 and tokens.shape == logp.shape == u.shape
    zs, us = z.double().cpu().numpy(), u.double().cpu().numpy()
    for b in range(len(us)):
        t, l, near = reference_row(zs[b], us[b], **{k: per_row(v, b) for k, v in limits.items()})
        assert near > clear, f"row {b}: a border {near:.2g} away: another seed"
        assert tokens[b].item() == t, (b, tokens[b].item(), t, near)
        assert logp[b].item() == l or abs(logp[b].item() - l) <= 2.0 ** -24 * abs(l) + 2.0 ** -40, (b, logp[b].item(), l)
    return tokens, logp


def _logits(dtype, B, V, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, V, generator=g) * spread).to(dtype).cuda(), torch.rand(B, generator=g).cuda()


LIMITS = [dict(), dict(temperature=0.7), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.3, top_k=40, top_p=0.8, min_p=0.02),
          dict(temperature=0.5, top_p=0.5, min_p=0.1), dict(top_k=3000, top_p=0.999), dict(top_k=1), dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("limits", LIMITS, ids=lambda d: "-".join(f"{k}{v}" for k, v in d.items()) or "none")
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("V", [1, 2, 30, 257, 4096, 4097, 32000])
def test_tokens_and_log_probabilities(V, dtype, limits):
    z, u = _logits(dtype, 6, V, seed=V)
    _check(z, u, **limits)


@pytest.mark.gpu
@pytest.mark.parametrize("limits", [dict(), dict(top_p=0.95), dict(top_k=50, top_p=0.9), dict(top_k=60000), dict(temperature=1e-4), dict(temperature=50.0, top_p=0.7),
                                    dict(top_k=20000, top_p=0.9, min_p=1e-4)], ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_large_vocabulary(dtype, limits):
    z, u = _logits(dtype, 3, 131003, seed=3)
    _check(z, u, **limits)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [30, 5000, 40000])
def test_equal_logits(V):
    """Ties go to the lowest index: all logits equal, two values, and a flat head longer than any list."""
    u = torch.tensor([0.0, 0.2, 0.5, 0.77, 0.999, 2 ** -24 * (2 ** 24 - 1)], device="cuda")
    flat = torch.zeros(6, V, device="cuda")
    two = (torch.arange(V, device="cuda") % 3 == 1).float().repeat(6, 1) * 2
    signed = torch.where(torch.arange(V, device="cuda") % 2 == 0, -0.0, 0.0).repeat(6, 1)
    for z in (flat, two, signed, flat.bfloat16()):
        for limits in (dict(top_k=7), dict(top_k=V // 2 + 1), dict(top_p=0.3), dict(top_p=0.61, top_k=V - 1), dict(min_p=1.0, top_p=0.9), dict(top_k=1), dict()):
            _check(z, u, clear=-1.0, **limits)      # (borders are met exactly here, by both sides)
    assert torch.equal(sample_tokens(signed, u, top_k=5)[0], sample_tokens(flat, u, top_k=5)[0])


@pytest.mark.gpu
def test_flat_and_peaked_rows():
    """Temperatures that put the whole row into one bin of the search, and rows whose mass is one candidate's."""
    z, u = _logits(torch.float32, 5, 20001, seed=11)
    for limits in (dict(temperature=1e4, top_p=0.37), dict(temperature=1e4, top_k=9000, top_p=0.37), dict(temperature=1e-3, top_p=0.99), dict(temperature=300.0, top_k=15000)):
        _check(z, u, **limits)
    z[:, 777] = 80.0
    _check(z, u, top_p=0.5)
    _check(z, u, top_k=3)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [9, 300, 9000])
def test_masked_and_infinite_logits(V):
    z, u = _logits(torch.float32, 8, V, seed=12)
    z[0, :] = -math.inf
    z[1, :] = math.nan
    z[2, 1:] = -math.inf
    z[3, ::2] = math.nan
    z[4, 3] = math.inf
    z[5, 2::3] = math.inf
    z[6, 1::2] = torch.finfo(torch.float32).min
    z[7, 1::2] = -math.inf
    for limits in (dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=V - 1, top_p=0.9, min_p=0.01), dict(temperature=0.0)):
        tokens, logp = _check(z, u, **limits)
        assert tokens[0] == -1 and tokens[1] == -1 and tokens[2] == 0 and tokens[4] == 3


@pytest.mark.gpu
def test_limits_by_row_and_views():
    B, V = 9, 3001
    z, u = _logits(torch.bfloat16, B, V, seed=13)
    g = torch.Generator().manual_seed(1)
    t = (torch.rand(B, generator=g) + 0.4).cuda()
    t[0] = 0.0
    k = torch.tensor([0, 1, 5, 100, 3000, 3001, 10 ** 6, 2, 50]).cuda()
    p = torch.tensor([1.0, 0.5, 0.9, 0.3, 0.95, 1.0, 0.7, 0.99, 0.0]).cuda()
    m = torch.tensor([0.0, 0.1, 0.01, 0.0, 0.2, 1.0, 0.0, 0.5, 0.0]).cuda()
    want = _check(z, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert torch.equal(sample_tokens(z, u, t, k.int(), p.double().float(), m)[0], want[0])
    for b in range(B):
        one = sample_tokens(z[b:b + 1], u[b:b + 1], t[b].item(), k[b].item(), p[b].item(), m[b].item())
        assert one[0][0] == want[0][b] and one[1][0] == want[1][b], b
    wide = torch.zeros(B, V + 5, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:-2] = z
    for view in (wide[:, 3:-2], z.t().contiguous().t(), z.float()):
        got = sample_tokens(view, u, t, k, p, m)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    off = sample_tokens(z, u, 1.0, torch.full((B,), -3, device="cuda"), torch.full((B,), math.nan, device="cuda"), torch.full((B,), -1.0, device="cuda"))
    assert torch.equal(off[0], sample_tokens(z, u)[0])
    assert sample_tokens(z[:0], u[:0])[0].shape == (0,)


@pytest.mark.gpu
def test_random_numbers_at_the_ends():
    z, _ = _logits(torch.float32, 6, 100, seed=14)
    z[:, 0], z[:, -1] = -math.inf, -200.0
    u = torch.tensor([0.0, -1.0, math.nan, 1.0, 5.0, 1 - 2 ** -24], device="cuda")
    tokens, _ = sample_tokens(z, u)
    assert tokens.tolist() == [1, 1, 1, 98, 98, 98]


@pytest.mark.gpu
def test_frequencies():
    """20000 draws of one row: every class within 5 standard deviations of its probability (1 in 10^6 per class for sound draws)."""
    n = 20000
    z = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5]).cuda()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    p = torch.softmax(z.double(), 0)
    counts = torch.bincount(sample_tokens(z.expand(n, 5), u.float())[0], minlength=5)
    assert ((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


@pytest.mark.gpu
def test_streams_graphs_and_repeats():
    z, u = _logits(torch.bfloat16, 7, 40000, seed=15)
    step = lambda: sample_tokens(z, u, 0.9, 50, 0.9, 0.01) + sample_tokens(z, u, 1.0, 0, 0.95)      # noqa: E731
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
        u.copy_(torch.rand(7, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(step(), held):
            assert torch.equal(a, b), i


@pytest.mark.gpu
def test_speller_sample():
    """The loop over ``forward_step``: temperature 0 is the Speller's own arg-max decode; a drawn sequence is what the log-probabilities of its
    own steps give."""
    c = synth.CONFIGS["tiny"]
    sd = synth.make_state_dict(synth.config_shapes("tiny"), seed=17)
    las = build_las(c, sd, max_label_len=6)
    x = torch.from_numpy(synth.make_inputs(3, 32, c["F"], seed=17)).cuda()
    with torch.no_grad():
        feat = las.listener(x)
        preds, _ = las.speller(feat)
    want = torch.stack(preds, 1)
    tokens, logprob = las.speller.sample(feat, torch.rand(6, 3, device="cuda"), temperature=0.0)
    assert torch.equal(tokens, want.argmax(-1)) and not logprob.any()
    u = torch.rand(6, 3, generator=torch.Generator().manual_seed(2)).cuda()
    tokens, logprob = las.speller.sample(feat, u, temperature=0.8, top_k=12, top_p=0.95)
    context, state, symbol = feat[:, 0], None, torch.zeros(3, dtype=torch.int64, device="cuda")
    for s in range(6):
        word = torch.cat([torch.nn.functional.one_hot(symbol, c["V"]).float(), context], -1)
        with torch.no_grad():
            logits, state, context, _ = las.speller.forward_step(word[:, None], state, feat)
        _check(logits, u[s], temperature=0.8, top_k=12, top_p=0.95)
        symbol = tokens[:, s]
        assert torch.equal(symbol, sample_tokens(logits, u[s], 0.8, 12, 0.95)[0])
    with pytest.raises(RuntimeError, match="uniforms"):
        las.speller.sample(feat, u[:, :2])


@pytest.mark.gpu
def test_refusals():
    z, u = _logits(torch.float32, 3, 20, seed=0)
    rows = torch.ones(3, device="cuda")
    for args, kw, message in [
        ((z.cpu(), u), {}, "no CPU fallback"), ((z[0], u), {}, "B,V"), ((z.double(), u), {}, "fp32, bf16 or fp16"), ((z[:, :0], u), {}, "B,V"),
        ((z, u[:2]), {}, "uniforms"), ((z, u.double()), {}, "uniforms"), ((z, u.cpu()), {}, "uniforms"),
        ((z, u), dict(temperature=-1.0), "temperature"), ((z, u), dict(temperature=math.nan), "temperature"), ((z, u), dict(temperature=math.inf), "temperature"),
        ((z, u), dict(top_k=-1), "top_k"), ((z, u), dict(top_p=1.5), "top_p"), ((z, u), dict(top_p=-0.1), "top_p"), ((z, u), dict(min_p=1.1), "min_p"),
        ((z, u), dict(min_p=math.nan), "min_p"), ((z, u), dict(temperature=rows[:2]), "temperature"), ((z, u), dict(top_k=rows), "top_k"),
        ((z, u), dict(top_p=rows.int()), "top_p"), ((z, u), dict(min_p=rows.cpu()), "min_p"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            sample_tokens(*args, **kw)


def test_c_entry_refuses_before_it_launches():
    """Status 1 and a message, nothing touched (runs without a GPU)."""
    L = _cabi.lib()
    good = dict(z=4096, sb=8, dtype=0, B=1, V=8, u=4096, t=1.0, k=0, p=1.0, m=0.0, tr=None, kr=None, pr=None, mr=None, tokens=4096, logp=None, work=None, stream=None)
    for change in (dict(z=None), dict(u=None), dict(tokens=None), dict(dtype=3), dict(dtype=-1), dict(B=-1), dict(V=0), dict(V=1 << 30), dict(V=1 << 16)):
        assert L.las_sample_tokens(*{**good, **change}.values()) == 1, change
        assert b"sampling" in L.las_last_error()
    assert L.las_sample_tokens(*{**good, "B": 0}.values()) == 0
    assert L.las_sample_workspace_bytes(1, 1 << 16) > 0 and L.las_sample_workspace_bytes(1, 64) == 0 and L.las_sample_workspace_bytes(1000, 1 << 16) == 0
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        sample_tokens(torch.zeros(2, 5), torch.zeros(2))


def test_reference_on_small_cases():
    """The definition by hand: weights 4, 2, 1, 1 in falling order 2, 0, 1, 3."""
    z = np.log([2.0, 1.0, 4.0, 1.0])
    row = lambda u, **k: reference_row(z, u, **k)[0]      # noqa: E731
    assert [row(u) for u in (0.0, 0.2, 0.26, 0.4, 0.9)] == [0, 0, 1, 2, 3]
    assert [row(u, top_k=3) for u in (0.0, 0.3, 0.5, 0.99)] == [0, 1, 2, 2]      # the tie of 1 and 3 goes to 1
    assert [row(u, top_p=0.4) for u in (0.0, 0.99)] == [2, 2]
    assert [row(u, top_p=0.7) for u in (0.0, 0.3, 0.4, 0.99)] == [0, 0, 2, 2]
    assert [row(u, min_p=0.3) for u in (0.1, 0.5)] == [0, 2]
    assert row(0.7, temperature=0.0) == 2 and row(0.7, top_k=1) == 2
