"""Timed cases of the decoder operators that stand beside the Speller's own: attention of decoder states over a Listener's
features (training step, forward, one decode step), distillation from a teacher's top logits (loss and gradient), and drawing
a token from logits.

``own`` False: plain torch forms of the formulas, in 32 bits (the sampler in 64: its answer hangs on borders of long sums), rounded
once at the end.  ``own`` True: the calls a program makes of the package.  ``exact``: the definitions in 64 bits, written apart."""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# --------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------
def listed():
    return [
        # a decoder with four heads over the paper-size Listener: 32 utterances of 800 frames (T' = 100), 128 characters
        dict(name="attend train 32x128 over 100", op="train", type="fp32", B=32, U=128, T=100, H=4, Hkv=4, D=128),
        # the long-utterance batch (3000 frames, T' = 375) in 16 bits
        dict(name="attend train 8x128 over 375", op="train", type="bf16", B=8, U=128, T=375, H=8, Hkv=8, D=64),
        # a large training batch with four query heads to a key head
        dict(name="attend train 16x512 over 1500", op="train", type="bf16", B=16, U=512, T=1500, H=16, Hkv=4, D=64),
        # scoring given transcripts against long recordings, no gradient; ragged sizes
        dict(name="attend 4x333 over 2999", op="attend", type="fp32", B=4, U=333, T=2999, H=8, Hkv=8, D=64),
        # one decode step of a validation batch: latency
        dict(name="one token 32 over 375", op="attend", type="bf16", B=32, U=1, T=375, H=8, Hkv=8, D=64),
        # one decode step over hours of sound: the features of 16 streams are read once
        dict(name="one token 16 over 30000", op="attend", type="fp16", B=16, U=1, T=30000, H=16, Hkv=4, D=128),
        # a character model taught by a larger one: the Speller's own vocabulary
        dict(name="distill characters", op="distill", type="fp32", B=32, U=128, V=30, K=8),
        # subword vocabulary, odd sizes
        dict(name="distill 5003 subwords", op="distill", type="fp32", B=16, U=201, V=5003, K=32),
        # a large vocabulary in 16 bits: logits read and their gradient written once
        dict(name="distill 128000 tokens", op="distill", type="bf16", B=8, U=512, V=128000, K=64),
        # one step of the Speller's batch
        dict(name="sample characters", op="sample", type="fp32", B=32, V=30, top_k=0, top_p=0.9, min_p=0.02, temperature=0.8, per_row=False),
        # a serving batch with all filters, each row its own temperature
        dict(name="sample 64 of 32000", op="sample", type="bf16", B=64, V=32000, top_k=50, top_p=0.9, min_p=0.01, temperature=0.5, per_row=True),
        # one row of a large vocabulary, no limit on the candidates but their mass
        dict(name="sample 1 of 128000", op="sample", type="fp32", B=1, V=128000, top_k=0, top_p=0.95, min_p=0.0, temperature=1.0, per_row=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = work(max(listed(), key=lambda c: max(work(c)["bytes"], work(c)["flops"] / 50)))
    most = max(most["bytes"], most["flops"] / 50) / 2
    while True:
        op = rng.choice(["train", "attend", "token", "distill", "sample"])
        if op in ("train", "attend", "token"):
            Hkv = rng.choice([1, 2, 4, 8])
            c = dict(op="train" if op == "train" else "attend", type=rng.choice(["fp32", "bf16", "bf16", "fp16"]),
                     B=_log(rng, 1, 32 if op != "token" else 64), U=1 if op == "token" else _log(rng, 2, 512),
                     T=_log(rng, 16, 2000 if op != "token" else 30000), H=Hkv * rng.choice([1, 1, 2, 4]), Hkv=Hkv,
                     D=rng.choice([32, 64, 64, 96, 128]))
        elif op == "distill":
            V = _log(rng, 30, 128000)
            c = dict(op="distill", type=rng.choice(["fp32", "bf16", "fp16"]), B=_log(rng, 1, 32), U=_log(rng, 1, 512), V=V, K=min(V, _log(rng, 1, 128)))
        else:
            V = _log(rng, 30, 128000)
            c = dict(op="sample", type=rng.choice(["fp32", "bf16", "fp16"]), B=_log(rng, 1, 256), V=V, top_k=rng.choice([0, 1, _log(rng, 2, 200)]),
                     top_p=rng.choice([1.0, 0.5, 0.9, 0.95]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), temperature=rng.choice([0.6, 1.0, 1.3]), per_row=rng.choice([False, True]))
        w = work(c)
        # (a plain form's time goes by its products in 32 bits too)
        if max(w["bytes"], w["flops"] / 50) <= most:
            return c


def _lengths(most, n):
    """n ragged lengths between half of `most` and all of it: the same numbers whatever the seed, which only deals them out."""
    return [max(1, most - (most // 2) * i // max(1, n)) for i in range(n)]


def work(case):
    c = case
    size = 4 if c["type"] == "fp32" else 2
    if c["op"] in ("train", "attend"):
        keys = sum(_lengths(c["T"], c["B"]))
        q, kv = c["B"] * c["U"] * c["H"] * c["D"] * size, keys * c["Hkv"] * c["D"] * size
        product = 2 * c["U"] * keys * c["H"] * c["D"]
        if c["op"] == "attend":
            return {"bytes": 2 * q + 2 * kv, "flops": 2 * product}
        # forward: q, k, v in, the output out; backward: those and the output's gradient in, three gradients out (dk and dv whole)
        whole = c["B"] * c["T"] * c["Hkv"] * c["D"] * size
        return {"bytes": 4 * q + 2 * kv + 2 * whole, "flops": 7 * product}
    if c["op"] == "distill":
        rows = sum(_lengths(c["U"], c["B"]))
        return {"bytes": rows * c["V"] * size + c["B"] * c["U"] * c["V"] * size + rows * c["K"] * (8 + size), "flops": 6 * rows * c["V"]}
    return {"bytes": c["B"] * c["V"] * size, "flops": 4 * c["B"] * c["V"]}


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = dict(case)
    dev, t = "cuda", TYPES[c["type"]]
    g = torch.Generator(device=dev).manual_seed(int(seed))
    rand = lambda *s, dtype=t: torch.randn(*s, device=dev, generator=g, dtype=torch.float32).to(dtype)      # noqa: E731
    deal = lambda most, n: torch.tensor(_lengths(most, n), dtype=torch.int32, device=dev)[torch.randperm(n, device=dev, generator=g)]      # noqa: E731
    B = c["B"]
    if c["op"] in ("train", "attend"):
        U, T, H, Hkv, D = (c[k] for k in ("U", "T", "H", "Hkv", "D"))
        s = dict(case=c, q=rand(B, U, H, D), k=rand(B, T, Hkv, D), v=rand(B, T, Hkv, D), lengths=deal(T, B))
        if c["op"] == "train":
            s["dout"] = rand(B, U, H, D)
            for n in "qkv":
                s[n].requires_grad_(True)
        return s
    if c["op"] == "distill":
        U, V, K = c["U"], c["V"], c["K"]
        # distinct indices in every row: a random start and steps of a random stride, which leaves no index twice below V
        start = torch.randint(0, V, (B, U, 1), device=dev, generator=g)
        stride = torch.randint(1, max(2, V // K + 1), (B, U, 1), device=dev, generator=g)
        index = (start + stride * torch.arange(K, device=dev)) % V
        teacher = (torch.sort(torch.randn(B, U, K, device=dev, generator=g) * 2, -1, descending=True).values + 4).to(t)
        logits = torch.randn(B, U, V, device=dev, generator=g).mul_(2)
        logits = logits.scatter_add_(2, index, 0.7 * teacher.float()).to(t).requires_grad_(True)      # a student that has learned something
        return dict(case=c, logits=logits, index=index, teacher=teacher, lengths=deal(U, B), temperature=2.0)
    V = c["V"]
    logits = rand(B, V, dtype=torch.float32).mul_(2.5).to(t)
    temperature = c["temperature"]
    if c["per_row"]:
        temperature = temperature + torch.rand(B, device=dev, generator=g)
    return dict(case=c, logits=logits, uniforms=torch.rand(B, device=dev, generator=g), temperature=temperature)


# --------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------
def _plain_attention(q, k, v, lengths, dout=None):
    B, U, H, D = q.shape
    T, Hkv = k.shape[1], k.shape[2]
    rows = lambda x: x.float().view(B, U, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)      # noqa: E731
    back = lambda x: x.view(B, Hkv, H // Hkv, U, D).permute(0, 3, 1, 2, 4).reshape(B, U, H, D).to(q.dtype)      # noqa: E731
    cols = lambda x: x.float().permute(0, 2, 1, 3).contiguous()      # noqa: E731
    scale = 1.0 / math.sqrt(D)
    Q, K, V = rows(q), cols(k), cols(v)
    keep = (torch.arange(T, device=q.device) < lengths[:, None])[:, None, None, :]
    s = torch.matmul(Q * scale, K.transpose(2, 3)).masked_fill_(~keep, -torch.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    del s
    o = torch.matmul(p, V)
    if dout is None:
        return back(o)
    dO = rows(dout)
    dv = torch.matmul(p.transpose(2, 3), dO)
    ds = torch.matmul(dO, V.transpose(2, 3)).sub_((dO * o).sum(-1, keepdim=True)).mul_(p)
    del p
    dq = torch.matmul(ds, K) * scale
    dk = torch.matmul(ds.transpose(2, 3), Q) * scale
    out = lambda x: x.permute(0, 2, 1, 3).contiguous().to(k.dtype)      # noqa: E731
    return back(o), back(dq), out(dk), out(dv)


def _plain_distill(logits, index, teacher, lengths, tau):
    """Mean over utterances of the mean over their steps of tau^2 KL(teacher's top entries || student), and its gradient."""
    B, U, V = logits.shape
    z = logits.float() / tau
    z -= z.amax(-1, keepdim=True)
    lse = z.exp().sum(-1, keepdim=True).log()
    t = teacher.float() / tau
    t = t - t.amax(-1, keepdim=True)
    logp = t - t.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    kl = (p * (logp - (z.gather(-1, index) - lse))).sum(-1)
    valid = torch.arange(U, device=z.device) < lengths[:, None]
    weight = torch.where(valid, 1.0 / (B * lengths[:, None].float()), 0.0)
    loss = (weight * kl).sum() * tau * tau
    grad = z.sub_(lse).exp_().scatter_add_(-1, index, -p).mul_((tau * weight)[..., None])
    return loss, grad.to(logits.dtype)


def _plain_sample(logits, uniforms, temperature, top_k, top_p, min_p):
    B, V = logits.shape
    t = temperature.double()[:, None] if torch.is_tensor(temperature) else float(temperature)
    x = logits.double() / t
    w = (x - x.amax(-1, keepdim=True)).exp()
    ws, order = torch.sort(w, dim=-1, descending=True, stable=True)
    rank = torch.arange(V, device=x.device)
    keep = rank < (top_k if top_k > 0 else V)
    ws = ws * keep
    before = ws.cumsum(-1) - ws
    keep = keep & (before < top_p * ws.sum(-1, keepdim=True)) & (ws >= min_p)
    w = torch.zeros_like(w).scatter_(-1, order, ws * keep)
    cum = w.cumsum(-1)
    token = (cum <= uniforms.double()[:, None] * cum[:, -1:]).sum(-1)
    return token, (w.gather(-1, token[:, None]) / cum[:, -1:]).log().squeeze(-1).float()


def run(state):
    s = state
    c = s["case"]
    if c["op"] in ("train", "attend"):
        if own:
            from las_pytorch_amd import cross_attention
            if c["op"] == "attend":
                return cross_attention(s["q"], s["k"], s["v"], s["lengths"])
            out = cross_attention(s["q"], s["k"], s["v"], s["lengths"])
            return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))
        with torch.no_grad():
            return _plain_attention(s["q"], s["k"], s["v"], s["lengths"], s.get("dout"))
    if c["op"] == "distill":
        if own:
            from las_pytorch_amd.solver.solver import distillation_loss_device
            loss = distillation_loss_device(s["logits"], s["index"], s["teacher"], s["temperature"], s["lengths"])
            return loss.detach(), *torch.autograd.grad(loss, (s["logits"],))
        with torch.no_grad():
            return _plain_distill(s["logits"], s["index"], s["teacher"], s["lengths"], s["temperature"])
    if own:
        from las_pytorch_amd import sample_tokens
        return sample_tokens(s["logits"], s["uniforms"], s["temperature"], c["top_k"], c["top_p"], c["min_p"])
    return _plain_sample(s["logits"], s["uniforms"], s["temperature"], c["top_k"], c["top_p"], c["min_p"])


# --------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("train", "attend"):
        return _exact_attention(s)
    if case["op"] == "distill":
        return _exact_distill(s)
    return _exact_sample(s)


def _exact_attention(s):
    """One utterance at a time, its valid keys alone; the gradients by autograd."""
    train = "dout" in s
    leaves = [s[n].detach().double().requires_grad_(train) for n in "qkv"]
    q, k, v = leaves
    share = q.shape[2] // k.shape[2]
    outs = []
    for b, n in enumerate(s["lengths"].tolist()):
        kb, vb = (x[b, :n].repeat_interleave(share, 1) for x in (k, v))
        a = torch.softmax(torch.einsum("uhd,thd->hut", q[b], kb) / math.sqrt(q.shape[-1]), -1)
        outs.append(torch.einsum("hut,thd->uhd", a, vb))
    out = torch.stack(outs)
    if not train:
        return out
    return (out.detach(), *torch.autograd.grad(out, leaves, s["dout"].double()))


def _exact_distill(s):
    """One utterance at a time, by log-softmax and autograd."""
    z, tau = s["logits"].detach(), float(s["temperature"])
    loss, grad = 0.0, []
    for b, n in enumerate(s["lengths"].tolist()):
        zb = z[b].double().requires_grad_(True)
        target = torch.softmax(s["teacher"][b, :n].double() / tau, -1)
        logq = torch.log_softmax(zb[:n] / tau, -1).gather(-1, s["index"][b, :n])
        part = tau * tau * (target * (target.log() - logq)).sum() / (n * z.shape[0])
        grad.append(torch.autograd.grad(part, zb)[0])
        loss = loss + part.detach()
        del zb, logq, part
    return loss, torch.stack(grad)


def _exact_sample(s):
    """Row by row: candidates in falling order, the shortest head that the three limits leave, then the inverse distribution."""
    c = s["case"]
    logits, u = s["logits"].double().cpu().numpy(), s["uniforms"].double().cpu().numpy()
    B, V = logits.shape
    temperature = s["temperature"].double().cpu().numpy() if torch.is_tensor(s["temperature"]) else np.full(B, float(s["temperature"]))
    tokens, logp = np.zeros(B, np.int64), np.zeros(B)
    for b in range(B):
        x = logits[b] / temperature[b]
        order = np.argsort(-x, kind="stable")[:c["top_k"] or V]
        e = np.exp(x[order] - x[order[0]])
        head = int(np.searchsorted(np.cumsum(e), c["top_p"] * e.sum(), side="left")) + 1
        head = min(head, int((e >= c["min_p"]).sum()))
        kept = np.sort(order[:head])
        e = np.exp(x[kept] - x[order[0]])
        at = min(int(np.searchsorted(np.cumsum(e), u[b] * e.sum(), side="right")), head - 1)
        tokens[b], logp[b] = kept[at], np.log(e[at] / e.sum())
    return torch.from_numpy(tokens), torch.from_numpy(logp)
