"""Measured cases of the preference-tuning operators: token log-probabilities
from hidden states (and their gradient), the paired preference loss, the
clipped policy loss with a KL term (each with its gradient) and the Muon update
of adapter matrices.

own = False computes every operator in plain torch operations; own = True makes
the calls a user makes of libllmcu.so through llm.cu_b200/llmcu.py.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

HIDDEN, VOCAB = 2048, 151936  # Qwen3-1.7B: the model this repository trains
MUON = (3.4445, -4.7750, 2.0315)  # a, b, c of the quintic Newton-Schulz step


def binding():
    """llm.cu_b200/llmcu.py (the directory's name is not a package name)."""
    if "llmcu" not in sys.modules:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.cu_b200", "llmcu.py")
        spec = importlib.util.spec_from_file_location("llmcu", path)
        sys.modules["llmcu"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["llmcu"])
    return sys.modules["llmcu"]


# ------------------------------------------------------------------- cases
def listed():
    return [
        # scoring the one token just chosen; the step's batch (8 x 512); an odd batch of the tiny model
        {"name": "logprobs one token", "op": "logprobs", "rows": 1, "hidden": HIDDEN, "vocab": VOCAB},
        {"name": "logprobs 8x512", "op": "logprobs", "rows": 4096, "hidden": HIDDEN, "vocab": VOCAB},
        {"name": "logprobs tiny odd", "op": "logprobs", "rows": 333, "hidden": 256, "vocab": 4096},
        # the same in the backward direction: the step's batch, and one short ragged sequence
        {"name": "logprobs_bwd 8x512", "op": "logprobs_bwd", "rows": 4096, "hidden": HIDDEN, "vocab": VOCAB},
        {"name": "logprobs_bwd 130", "op": "logprobs_bwd", "rows": 130, "hidden": HIDDEN, "vocab": VOCAB},
        # the pairs of one step on one GPU; a large batch of long pairs whose rows are padded
        {"name": "preference 4x512", "op": "preference", "kind": "sigmoid", "pairs": 4, "seq": 512, "pad": 0,
         "beta": 0.1, "smoothing": 0.0, "margin": 0.0, "mean_tokens": False, "ref": True},
        {"name": "preference 256x4095", "op": "preference", "kind": "sigmoid", "pairs": 256, "seq": 4095, "pad": 9,
         "beta": 0.3, "smoothing": 0.1, "margin": 0.5, "mean_tokens": False, "ref": True},
        # a step's samples with one advantage each; ragged groups with per-token advantages and no reference
        # model; a large rollout batch with every term
        {"name": "policy 8x512", "op": "policy", "batch": 8, "seq": 512, "pad": 0, "agg": "token_mean", "beta": 0.04,
         "clip_low": 0.2, "clip_high": 0.2, "dual": 0.0, "ref": True, "token_adv": False},
        {"name": "policy 64x2047", "op": "policy", "batch": 64, "seq": 2047, "pad": 1, "agg": "sequence_mean",
         "beta": 0.0, "clip_low": 0.2, "clip_high": 0.28, "dual": 0.0, "ref": False, "token_adv": True},
        {"name": "policy 1024x8192", "op": "policy", "batch": 1024, "seq": 8192, "pad": 0, "agg": "constant",
         "beta": 0.01, "clip_low": 0.2, "clip_high": 0.28, "dual": 3.0, "ref": True, "token_adv": True},
        # every rank-16 A matrix of the 28 layers' four attention adapters; a few odd B matrices
        {"name": "muon 112x16x2048", "op": "muon", "count": 112, "rows": 16, "cols": 2048, "nesterov": True,
         "match_rms": False},
        {"name": "muon 4x1023x7", "op": "muon", "count": 4, "rows": 1023, "cols": 7, "nesterov": True,
         "match_rms": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs_bwd", "preference", "policy", "muon"])
    if op in ("logprobs", "logprobs_bwd"):
        return {"op": op, "rows": _log(rng, 1, 4096), "hidden": 8 * _log(rng, 8, HIDDEN // 8),
                "vocab": 8 * _log(rng, 16, VOCAB // 8)}
    if op == "preference":
        pairs = _log(rng, 1, 256)
        return {"op": op, "kind": rng.choice(["sigmoid", "hinge", "squared"]), "pairs": pairs,
                "seq": _log(rng, 1, min(32768, 1048576 // pairs)), "pad": rng.choice([0, 0, 1, 8]),
                "beta": round(rng.uniform(0.05, 0.5), 3), "smoothing": 0.0, "margin": 0.0,
                "mean_tokens": rng.random() < 0.4, "ref": rng.random() < 0.7}
    if op == "policy":
        batch = _log(rng, 1, 1024)
        ref = rng.random() < 0.6
        return {"op": op, "batch": batch, "seq": _log(rng, 1, min(32768, 8388608 // batch)),
                "pad": rng.choice([0, 0, 1, 8]), "agg": rng.choice(["token_mean", "sequence_mean", "constant"]),
                "beta": 0.04 if ref else 0.0, "clip_low": 0.2, "clip_high": rng.choice([0.2, 0.28]),
                "dual": rng.choice([0.0, 3.0]), "ref": ref, "token_adv": rng.random() < 0.5}
    rank, side = rng.randint(1, 16), _log(rng, 16, 8192)
    rows, cols = (rank, side) if rng.random() < 0.5 else (side, rank)
    return {"op": op, "count": _log(rng, 1, min(112, 4194304 // (rank * side))), "rows": rows, "cols": cols,
            "nesterov": rng.random() < 0.7, "match_rms": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("logprobs", "logprobs_bwd"):
        M, H, V = case["rows"], case["hidden"], case["vocab"]
        s["E"] = torch.randn(V, H, generator=g, device=dev, dtype=torch.float16).mul_(0.9 / math.sqrt(H) * 1.0)
        s["targets"] = torch.randint(0, V, (M,), generator=g, device=dev, dtype=torch.int32)
        # normed hidden states that lean towards the target's row by differing amounts: probabilities of the
        # targets from about 1 / V to nearly 1
        lean = torch.rand(M, 1, generator=g, device=dev) * 16
        x = torch.randn(M, H, generator=g, device=dev) + lean * s["E"][s["targets"].long()].float()
        s["x"] = x.half()
        # prompt tokens are not scored (an eighth of the rows; the first row always is)
        skip = torch.rand(M, generator=g, device=dev) < 0.125
        skip[0] = False
        s["targets"][skip] = -1
        if op == "logprobs_bwd":
            s["lse"] = _lse(s["x"], s["E"])
            s["dlogp"] = torch.randn(M, generator=g, device=dev).masked_fill_(skip, 0.0) / M
            s["scale"] = 64.0 * M  # keeps the fp16 gradient in range
        return s
    if op == "preference":
        rows, seq = 2 * case["pairs"], case["seq"]
    elif op == "policy":
        rows, seq = case["batch"], case["seq"]
    if op in ("preference", "policy"):
        ld = seq + case["pad"]
        # completions: a prompt of some length in front, padding behind; where there are many rows one is empty
        pos = torch.arange(ld, device=dev)
        start = (torch.rand(rows, 1, generator=g, device=dev) * 0.3 * seq).long()
        end = seq - (torch.rand(rows, 1, generator=g, device=dev) * 0.4 * seq).long()
        mask = (pos >= start) & (pos < end)
        if rows >= 8:
            mask[5] = False
        logp = -torch.empty(rows, ld, device=dev).exponential_(0.8, generator=g)
        s["mask"] = mask
        noise = lambda sd: sd * torch.randn(rows, ld, generator=g, device=dev)  # noqa: E731
        # what is not scored holds nothing of use: -inf, as the log-probability of a banned token
        s["ref"] = (logp + noise(0.2)).masked_fill(~mask, float("-inf")) if case["ref"] else None
        if op == "policy":
            s["old"] = (logp + noise(0.15)).masked_fill(~mask, float("-inf"))
            shape = (rows, ld) if case["token_adv"] else (rows,)
            s["adv"] = torch.randn(*shape, generator=g, device=dev)
            s["norm"] = 0.7 * rows * seq
        s["logp"] = logp.masked_fill(~mask, float("-inf"))
        return s
    n, r, c = case["count"], case["rows"], case["cols"]
    k, m = min(r, c), max(r, c)
    # gradients with a spectrum that falls over two orders of magnitude, as low-rank adapters' do
    mix = torch.randn(n, k, k, generator=g, device=dev) * torch.logspace(0, -2, k, device=dev)
    grads = [torch.bmm(mix, torch.randn(n, k, m, generator=g, device=dev)) * 1e-3 for _ in range(2)]
    grads = [x if r <= c else x.transpose(1, 2) for x in grads]
    s["grad"] = grads[0].contiguous()
    s["momentum"] = (grads[1] * 5).contiguous()
    s["w"] = torch.randn(n, r, c, generator=g, device=dev) / math.sqrt(m)
    return s


def _lse(x, E):
    """log sum exp of the rows' logits, a thousand rows at a time."""
    return torch.cat([torch.logsumexp(p.float() @ E.float().t(), 1) for p in x.split(1024)])


# --------------------------------------------------------------------- run
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def plain_logprobs(s):
    logits = s["x"].float() @ s["E"].float().t()
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp().sum(1).log() + top[:, 0]
    t = s["targets"].long()
    picked = logits.gather(1, t.clamp(0)[:, None])[:, 0]
    return {"logp": torch.where(t >= 0, picked - lse, 0.0), "lse": lse}


def plain_logprobs_bwd(s):
    E = s["E"].float()
    d = (s["x"].float() @ E.t() - s["lse"][:, None]).exp().neg()
    t = s["targets"].long()
    rows = torch.arange(len(t), device=t.device)
    d[rows, t.clamp(0)] += 1.0
    g = torch.where(t >= 0, s["dlogp"] * s["scale"], 0.0)
    return {"dx": (g[:, None] * (d @ E)).half()}


def plain_preference(s):
    c = s["case"]
    P, S = c["pairs"], c["seq"]
    mask = s["mask"][:, :S]
    diff = s["logp"][:, :S].double()  # long sums that nearly cancel: in 64 bits
    if s["ref"] is not None:
        diff = diff - s["ref"][:, :S].double()
    total = torch.where(mask, diff, 0.0).sum(1)
    share = 1.0 / mask.sum(1).clamp(1) if c["mean_tokens"] else torch.ones_like(total)
    total = total * share
    D = total[:P] - total[P:]
    h = c["beta"] * D - c["margin"]
    if c["kind"] == "sigmoid":
        e = c["smoothing"]
        soft = lambda z: z.clamp(0) + torch.log1p(torch.exp(-z.abs()))  # noqa: E731  log(1 + e^z)
        loss = (1 - e) * soft(-h) + e * soft(h)
        dD = c["beta"] * (e - 1.0 / (1.0 + torch.exp(h)))
    elif c["kind"] == "hinge":
        loss = (1 - h).clamp(0)
        dD = torch.where(h < 1, -c["beta"], 0.0).double()
    else:
        off = D - 0.5 / c["beta"]
        loss, dD = off * off, 2 * off
    row = torch.cat([dD, -dD]) * share / P
    dlogp = torch.where(mask, row[:, None], 0.0).float()
    return {"loss": loss.float(), "reward": (c["beta"] * total).float(), "dlogp": dlogp}


def plain_policy(s):
    c = s["case"]
    B, S = c["batch"], c["seq"]
    mask = s["mask"][:, :S]
    lp = s["logp"][:, :S].double()  # differences and what lies next to the clip's borders: in 64 bits
    delta = lp - s["old"][:, :S].double()
    ratio = torch.exp(delta)
    adv = (s["adv"][:, :S] if c["token_adv"] else s["adv"][:, None]).double().expand(B, S)
    low, high = 1 - _f32(c["clip_low"]), 1 + _f32(c["clip_high"])
    clipped = ((adv > 0) & (ratio > high)) | ((adv < 0) & (ratio < low))
    obj = torch.where(clipped, ratio.clamp(low, high), ratio) * adv
    if c["dual"] > 0:
        capped = (adv < 0) & (ratio > c["dual"])
        obj = torch.where(capped, c["dual"] * adv, obj)
        clipped = clipped | capped
    loss, grad = -obj, torch.where(clipped, 0.0, -ratio * adv)
    kl = torch.zeros_like(lp)
    if s["ref"] is not None:
        d = s["ref"][:, :S].double() - lp
        up = torch.expm1(d)
        kl = up - d
        loss, grad = loss + _f32(c["beta"]) * kl, grad - _f32(c["beta"]) * up
    count = mask.sum(1)
    tokens = count.sum()
    if c["agg"] == "token_mean":
        weight = (1.0 / tokens.clamp(1).double()).expand(B)
    elif c["agg"] == "sequence_mean":
        weight = 1.0 / (count.clamp(1).double() * B)
    else:
        weight = torch.full((B,), 1.0 / s["norm"], dtype=torch.float64, device=lp.device)
    weight = weight[:, None]
    keep = lambda v: torch.where(mask, v, 0.0)  # noqa: E731
    n = tokens.clamp(1)
    return {"loss": (keep(loss) * weight).sum().float(), "kl": (keep(kl).sum() / n).float(),
            "clipped": (keep(clipped.double()).sum() / n).float(), "tokens": tokens.float(),
            "dlogp": (keep(grad) * weight).float()}


def _f32(v):
    """The value a 32-bit configuration field holds."""
    return float(torch.tensor(v, dtype=torch.float32))


LR, WD, MU, EPS = 1e-3, 0.01, 0.95, 1e-7


def plain_muon(s):
    c = s["case"]
    a, b, k = (_f32(v) for v in MUON)
    s["momentum"].mul_(MU).add_(s["grad"])
    u = s["grad"] + MU * s["momentum"] if c["nesterov"] else s["momentum"]
    x = u.double()  # five steps raise the small directions by hundreds: in 64 bits
    x = x if c["rows"] <= c["cols"] else x.transpose(1, 2)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)

    def step(x):
        A = x @ x.transpose(1, 2)
        return a * x + (b * A + k * (A @ A)) @ x

    x = step(step(step(step(step(x)))))
    x = x if c["rows"] <= c["cols"] else x.transpose(1, 2)
    scale = 0.2 * math.sqrt(max(c["rows"], c["cols"])) if c["match_rms"] else math.sqrt(max(1.0, c["rows"] / c["cols"]))
    s["w"].copy_(s["w"].double() * (1 - LR * WD) - LR * scale * x)
    return {"w": s["w"], "momentum": s["momentum"]}


_plain = {"logprobs": plain_logprobs, "logprobs_bwd": plain_logprobs_bwd, "preference": plain_preference,
          "policy": plain_policy, "muon": plain_muon}


# ------------------------------------------------------ the framework's calls
def _buffers(s, **shapes):
    """Outputs and workspace that a program keeps from step to step."""
    if "out" not in s:
        s["out"] = {k: torch.empty(shape, dtype=t, device="cuda") for k, (shape, t) in shapes.items()}
    return s["out"]


def own_logprobs(s):
    L, (M, H), V = binding(), s["x"].shape, len(s["E"])
    if "bytes" not in s:
        s["bytes"] = L.lm_logprobs_workspace(M, H, V, False)
    o = _buffers(s, logp=(M, torch.float32), lse=(M, torch.float32), ws=(s["bytes"], torch.uint8))
    L.lm_logprobs(s["x"].data_ptr(), s["E"].data_ptr(), s["targets"].data_ptr(), o["logp"].data_ptr(),
                  o["lse"].data_ptr(), M, H, V, H, H, o["ws"].data_ptr(), s["bytes"],
                  torch.cuda.current_stream().cuda_stream)
    return {"logp": o["logp"], "lse": o["lse"]}


def own_logprobs_bwd(s):
    L, (M, H), V = binding(), s["x"].shape, len(s["E"])
    if "bytes" not in s:
        s["bytes"] = L.lm_logprobs_workspace(M, H, V, True)
    o = _buffers(s, dx=((M, H), torch.float16), ws=(s["bytes"], torch.uint8))
    L.lm_logprobs_bwd(s["x"].data_ptr(), s["E"].data_ptr(), s["targets"].data_ptr(), s["lse"].data_ptr(),
                      s["dlogp"].data_ptr(), o["dx"].data_ptr(), M, H, V, H, H, H, s["scale"], o["ws"].data_ptr(),
                      s["bytes"], torch.cuda.current_stream().cuda_stream)
    return {"dx": o["dx"]}


def own_preference(s):
    L, c = binding(), s["case"]
    P, S, ld = c["pairs"], c["seq"], c["seq"] + c["pad"]
    if "cfg" not in s:
        kind = {"sigmoid": L.PREF_SIGMOID, "hinge": L.PREF_HINGE, "squared": L.PREF_SQUARED}[c["kind"]]
        s["cfg"] = L.Preference(kind, c["beta"], c["smoothing"], c["margin"], c["mean_tokens"])
    o = _buffers(s, loss=(P, torch.float32), reward=(2 * P, torch.float32), dlogp=((2 * P, ld), torch.float32))
    L.preference_loss(s["cfg"], s["logp"].data_ptr(), 0 if s["ref"] is None else s["ref"].data_ptr(),
                      s["mask"].data_ptr(), 0, o["loss"].data_ptr(), o["reward"].data_ptr(), o["dlogp"].data_ptr(),
                      P, S, ld, torch.cuda.current_stream().cuda_stream)
    return {"loss": o["loss"], "reward": o["reward"], "dlogp": o["dlogp"][:, :S]}


def own_policy(s):
    L, c = binding(), s["case"]
    B, S, ld = c["batch"], c["seq"], c["seq"] + c["pad"]
    if "cfg" not in s:
        agg = {"token_mean": L.POLICY_TOKEN_MEAN, "sequence_mean": L.POLICY_SEQUENCE_MEAN,
               "constant": L.POLICY_CONSTANT}[c["agg"]]
        s["cfg"] = L.Policy(c["clip_low"], c["clip_high"], c["beta"], c["dual"], agg, s["norm"], c["token_adv"])
        s["bytes"] = L.policy_loss_workspace(B, S)
    o = _buffers(s, stats=(4, torch.float32), dlogp=((B, ld), torch.float32), ws=(s["bytes"], torch.uint8))
    L.policy_loss(s["cfg"], s["logp"].data_ptr(), s["old"].data_ptr(), 0 if s["ref"] is None else s["ref"].data_ptr(),
                  s["adv"].data_ptr(), s["mask"].data_ptr(), o["stats"].data_ptr(), o["dlogp"].data_ptr(), B, S, ld,
                  o["ws"].data_ptr(), s["bytes"], torch.cuda.current_stream().cuda_stream)
    loss, kl, clipped, tokens = o["stats"].unbind()
    return {"loss": loss, "kl": kl, "clipped": clipped, "tokens": tokens, "dlogp": o["dlogp"][:, :S]}


def own_muon(s):
    L, c = binding(), s["case"]
    if "cfg" not in s:
        s["cfg"] = L.Muon(lr=LR, momentum=MU, weight_decay=WD, eps=EPS, nesterov=c["nesterov"],
                          match_rms=c["match_rms"])
    L.muon_update(s["cfg"], s["w"].data_ptr(), s["grad"].data_ptr(), s["momentum"].data_ptr(), c["count"], c["rows"],
                  c["cols"], torch.cuda.current_stream().cuda_stream)
    return {"w": s["w"], "momentum": s["momentum"]}


_own = {"logprobs": own_logprobs, "logprobs_bwd": own_logprobs_bwd, "preference": own_preference,
        "policy": own_policy, "muon": own_muon}


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("logprobs", "logprobs_bwd"):
        M, H, V = case["rows"], case["hidden"], case["vocab"]
        if op == "logprobs":
            return {"bytes": 2 * (M * H + V * H) + 12 * M, "flops": 2.0 * M * H * V}
        # the logits are formed again, then multiplied by the head
        return {"bytes": 2 * (2 * M * H + V * H) + 12 * M, "flops": 4.0 * M * H * V}
    if op == "preference":
        n = 2 * case["pairs"] * case["seq"]
        return {"bytes": n * (9 + (4 if case["ref"] else 0)) + 12 * case["pairs"], "flops": 4.0 * n}
    if op == "policy":
        n = case["batch"] * case["seq"]
        per = 13 + (4 if case["ref"] else 0) + (4 if case["token_adv"] else 0)
        return {"bytes": n * per + 4 * case["batch"], "flops": 20.0 * n}
    k, m = sorted((case["rows"], case["cols"]))
    n = case["count"]
    # the Gram matrix (symmetric) and one product with it of every element; five steps of k x k products
    return {"bytes": 20 * n * k * m, "flops": n * (k * (k + 1.0) * m + 2.0 * k * k * m + 8 * m * k + 40.0 * k ** 3)}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": exact_logprobs, "logprobs_bwd": exact_logprobs_bwd, "preference": exact_preference,
            "policy": exact_policy, "muon": exact_muon}[case["op"]](s)


def exact_logprobs(s):
    E, out = s["E"].double(), []
    for x, t in zip(s["x"].split(512), s["targets"].long().split(512)):
        z = torch.log_softmax(x.double() @ E.t(), 1)
        one = torch.where(t >= 0, z.gather(1, t.clamp(0)[:, None])[:, 0], 0.0)
        # any column tells lse: logit - log_softmax
        out.append((one, (x.double() * E[0]).sum(1) - z[:, 0]))
    return {"logp": torch.cat([o[0] for o in out]), "lse": torch.cat([o[1] for o in out])}


def exact_logprobs_bwd(s):
    E, out = s["E"].double(), []
    parts = [s[k].split(512) for k in ("x", "targets", "lse", "dlogp")]
    for x, t, lse, g in zip(*parts):
        p = torch.exp(x.double() @ E.t() - lse.double()[:, None])
        live = (t >= 0).double()[:, None]
        out.append(s["scale"] * g.double()[:, None] * live * (E[t.long().clamp(0)] - p @ E))
    return {"dx": torch.cat(out)}


def exact_preference(s):
    """By autograd of the loss in 64 bits."""
    c = s["case"]
    P, S = c["pairs"], c["seq"]
    mask = s["mask"][:, :S]
    lp = s["logp"][:, :S].double().masked_fill(~mask, 0.0).requires_grad_()
    z = lp * mask
    if s["ref"] is not None:
        z = z - s["ref"][:, :S].double().masked_fill(~mask, 0.0)
    R = z.sum(1) / (mask.sum(1).clamp(min=1) if c["mean_tokens"] else 1)
    D = R[:P] - R[P:]
    h = c["beta"] * D - c["margin"]
    if c["kind"] == "sigmoid":
        F = torch.nn.functional
        loss = -(1 - c["smoothing"]) * F.logsigmoid(h) - c["smoothing"] * F.logsigmoid(-h)
    elif c["kind"] == "hinge":
        loss = torch.relu(1 - h)
    else:
        loss = (D - 1 / (2 * c["beta"])) ** 2
    loss.mean().backward()
    return {"loss": loss.detach(), "reward": (c["beta"] * R).detach(), "dlogp": lp.grad}


def exact_policy(s):
    """By autograd of the loss in 64 bits, over the scored tokens alone."""
    c = s["case"]
    B, S = c["batch"], c["seq"]
    row, col = s["mask"][:, :S].nonzero(as_tuple=True)
    lp = s["logp"][row, col].double().requires_grad_()
    r = (lp - s["old"][row, col].double()).exp()
    A = (s["adv"][row, col] if c["token_adv"] else s["adv"][row]).double()
    lo, hi = 1 - _f32(c["clip_low"]), 1 + _f32(c["clip_high"])
    obj = torch.minimum(r * A, r.clamp(lo, hi) * A)
    cut = (r * A > r.clamp(lo, hi) * A)
    if c["dual"] > 0:
        cut = cut | ((A < 0) & (c["dual"] * A > obj))
        obj = torch.where(A < 0, torch.maximum(obj, c["dual"] * A), obj)
    kl = torch.zeros_like(A)
    if s["ref"] is not None:
        d = s["ref"][row, col].double() - lp
        kl = d.expm1() - d
    per = _f32(c["beta"]) * kl - obj
    n = len(row)
    count = torch.bincount(row, minlength=B).double()
    if c["agg"] == "token_mean":
        loss = per.sum() / max(n, 1)
    elif c["agg"] == "sequence_mean":
        loss = (per / count[row]).sum() / B
    else:
        loss = per.sum() / s["norm"]
    dlogp = torch.zeros(B, S, dtype=torch.float64, device=A.device)
    if n:
        loss.backward()
        dlogp[row, col] = lp.grad
    return {"loss": loss.detach(), "kl": kl.detach().sum() / max(n, 1), "clipped": cut.double().sum() / max(n, 1),
            "tokens": torch.tensor(float(n), dtype=torch.float64), "dlogp": dlogp}


def exact_muon(s):
    """By the singular values: each step maps v to a v + b v^3 + c v^5 and leaves the singular vectors."""
    c = s["case"]
    a, b, k = (_f32(v) for v in MUON)
    g, m = s["grad"].double().cpu(), s["momentum"].double().cpu()
    m = MU * m + g
    u = g + MU * m if c["nesterov"] else m
    U, S, Vh = torch.linalg.svd(u, full_matrices=False)
    v = S / (S.square().sum(1, keepdim=True).sqrt() + EPS)
    for _ in range(5):
        v = v * (a + b * v ** 2 + k * v ** 4)
    x = (U * v[:, None, :]) @ Vh
    scale = 0.2 * math.sqrt(max(c["rows"], c["cols"])) if c["match_rms"] else math.sqrt(max(1.0, c["rows"] / c["cols"]))
    return {"w": s["w"].double().cpu() * (1 - LR * WD) - LR * scale * x, "momentum": m}
