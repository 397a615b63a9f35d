"""Preference tuning on a training context against fp32 CPU autograd of the same
model (oracle/golden.py's layers) with the losses written out.

Tolerances are the step's: 1e-3 relative for losses and log-probabilities
(rel-L2), gradients rel-L2 <= 1e-2 and cosine >= 0.999."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

RTOL, GRAD_RELL2, GRAD_COS = 1e-3, 1e-2, 0.999


def token_logps(G, cfg, base, params, tokens, targets):
    """Log-probabilities [B, S] of the targets (0 where outside the vocabulary), differentiable in params."""
    W = {k: torch.from_numpy(v) for k, v in base.items()}
    cos, sin = G.rope_tables(cfg, tokens.shape[1])

    def lora_add(x, name):
        if name + ".A" not in params:
            return 0.0
        return (x @ params[name + ".A"].t() @ params[name + ".B"].t()) * cfg.lora_scale

    x, _ = G._layers(cfg, W, lora_add, tokens, cos, sin, False)
    logits = G.rmsnorm(x, W["final_norm"], cfg.rms_eps) @ W["embed"].t()
    t = torch.from_numpy(targets.astype(np.int64))
    ok = (t >= 0) & (t < cfg.vocab)
    lp = torch.log_softmax(logits, -1).gather(-1, t.clamp(0, cfg.vocab - 1)[..., None])[..., 0]
    return torch.where(ok, lp, 0.0), ok


class Case:
    """A context, its golden parameters and a batch whose prompts and paddings are not scored."""

    def __init__(self, llmcu, batch=4, seq=48, seed=3, lora_std=None, **run):
        from oracle import golden as G
        self.G, self.cfg = G, G.CFG_TINY
        cfg = self.cfg
        self.base = G.make_base_weights(cfg, seed, round_fp16=True)
        self.lora = G.make_lora(cfg, seed + 1)
        if lora_std == 0:
            for k in self.lora:
                if k.endswith(".B"):
                    self.lora[k][...] = 0
        self.tok, tgt = G.make_tokens(cfg, batch, seq, seed + 2)
        rng = np.random.Generator(np.random.PCG64(seed))
        self.tgt = tgt.copy()
        for b in range(batch):
            self.tgt[b, : rng.integers(0, seq // 3)] = -1
            self.tgt[b, seq - rng.integers(1, seq // 3):] = -100
        self.tgt[1] = -1  # nothing scored
        self.rng = rng
        self.ctx = llmcu.Context(llmcu.Model.tiny(), llmcu.Lora(cfg.lora_rank, cfg.lora_alpha),
                                 llmcu.Run(batch, seq, **run))
        self.ctx.set_base(self.base)
        self.ctx.set_lora_dict(self.lora)
        self.params = {k: torch.from_numpy(v).clone().requires_grad_(True) for k, v in self.lora.items()}

    def logps(self):
        return token_logps(self.G, self.cfg, self.base, self.params, self.tok, self.tgt)

    def check_grads(self, loss):
        loss.backward()
        got = self.ctx.grads_dict()
        for k, p in self.params.items():
            want = p.grad.numpy()
            r, c = self.G.rel_l2(got[k], want), self.G.cosine(got[k], want)
            assert r <= GRAD_RELL2 and c >= GRAD_COS, f"{k}: rel_l2 {r:.3e} cos {c:.6f}"


def test_score_matches_golden(llmcu, cuda_device):
    c = Case(llmcu)
    with torch.no_grad():
        want, ok = c.logps()
        base = token_logps(c.G, c.cfg, c.base, {}, c.tok, c.tgt)[0]
    got = c.ctx.score(c.tok, c.tgt)
    alone = c.ctx.score(c.tok, c.tgt, adapters=False)
    assert (got[~ok.numpy()] == 0).all() and (alone[~ok.numpy()] == 0).all()
    assert c.G.rel_l2(got, want.numpy()) <= RTOL and c.G.rel_l2(alone, base.numpy()) <= RTOL
    assert np.abs(got - alone).max() > 0.01  # the adapters matter
    assert np.array_equal(got, c.ctx.score(c.tok, c.tgt))
    c.ctx.close()


@pytest.mark.parametrize("targets", [0x0F, 0x7F])
def test_base_score_does_not_read_the_adapters(llmcu, cuda_device, targets):
    """Diverged adapters (NaN, infinite, past fp16's range) leave the reference model's score as it is."""
    from oracle import golden as G
    tok, tgt = G.make_tokens(G.CFG_TINY, 2, 40, 4)
    ctx = llmcu.Context(llmcu.Model.tiny(), llmcu.Lora(4, 8.0, targets), llmcu.Run(2, 40))
    ctx.init_base_synthetic(3)
    ctx.init_lora_synthetic(4)
    good = ctx.lora_dict()
    want = ctx.score(tok, tgt, adapters=False)
    assert np.isfinite(want).all()
    for bad in (np.nan, np.inf, 1e6):
        ctx.set_lora_dict({k: np.full_like(v, bad) for k, v in good.items()})
        assert np.array_equal(want, ctx.score(tok, tgt, adapters=False))
    ctx.set_lora_dict(good)
    assert np.isfinite(ctx.score(tok, tgt)).all()
    ctx.close()


def test_score_leaves_the_step_as_it_was(llmcu, cuda_device):
    """A cross-entropy step gives the same bits with and without a base-model score before it."""
    c = Case(llmcu, deterministic=True)
    tgt = np.abs(c.tgt) % c.cfg.vocab
    loss = c.ctx.forward_backward(c.tok, tgt)
    grads = c.ctx.grads_dict()
    c.ctx.score(c.tok, tgt, adapters=False)
    assert c.ctx.forward_backward(c.tok, tgt) == loss
    again = c.ctx.grads_dict()
    assert all(np.array_equal(grads[k], again[k]) for k in grads)
    c.ctx.close()


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("mean", [False, True])
def test_preference_step_matches_golden(llmcu, cuda_device, kind, mean):
    c = Case(llmcu, batch=6, seq=48, seed=7 + mean)
    ref = c.ctx.score(c.tok, c.tgt, adapters=False)
    k = {"sigmoid": llmcu.PREF_SIGMOID, "hinge": llmcu.PREF_HINGE, "squared": llmcu.PREF_SQUARED}[kind]
    beta = 0.1 if not mean else 2.0
    cfg = llmcu.Preference(k, beta, 0.05 if kind == "sigmoid" else 0.0, 0.0, mean)
    loss, rewards = c.ctx.preference_forward_backward(c.tok, c.tgt, cfg, ref)
    lp, ok = c.logps()
    z = lp - torch.from_numpy(ref) * ok
    R = (z * ok).sum(1) / (ok.sum(1).clamp(min=1) if mean else 1)
    P = len(R) // 2
    D = R[:P] - R[P:]
    h = beta * D
    F = torch.nn.functional
    if kind == "sigmoid":
        per = -0.95 * F.logsigmoid(h) - 0.05 * F.logsigmoid(-h)
    elif kind == "hinge":
        per = torch.relu(1 - h)
    else:
        per = (D - 1 / (2 * beta)) ** 2
    want = per.mean()
    assert abs(loss - want.item()) <= RTOL * abs(want.item()), (loss, want.item())
    # a reward sums dozens of log-probability differences, each off by 1e-3 of a log-probability at most
    assert np.abs(rewards - beta * R.detach().numpy()).max() <= beta * RTOL * lp.abs().sum(1).max().item()
    assert rewards[1] == 0
    c.check_grads(want)
    c.ctx.close()


@pytest.mark.parametrize("agg", [0, 1, 2])
@pytest.mark.parametrize("token_adv", [False, True])
def test_policy_step_matches_golden(llmcu, cuda_device, agg, token_adv):
    c = Case(llmcu, batch=5, seq=40, seed=20 + agg)
    B, S = c.tok.shape
    ref = c.ctx.score(c.tok, c.tgt, adapters=False)
    # samples of a policy near this one, none next to a border of the clip
    step = c.rng.choice([-0.5, -0.1, 0.0, 0.1, 0.5], size=(B, S)).astype(np.float32)
    old = c.ctx.score(c.tok, c.tgt) - step
    adv = c.rng.standard_normal((B, S) if token_adv else (B,)).astype(np.float32)
    cfg = llmcu.Policy(0.2, 0.3, 0.05, 0.0, agg, 100.0, token_adv)
    loss, stats = c.ctx.policy_forward_backward(c.tok, c.tgt, old, adv, cfg, ref)
    lp, ok = c.logps()
    A = torch.from_numpy(adv if token_adv else np.repeat(adv[:, None], S, 1))
    r = (lp - torch.from_numpy(old)).exp()
    obj = torch.minimum(r * A, r.clamp(0.8, 1.3) * A)
    d = torch.from_numpy(ref) - lp
    per = torch.where(ok, 0.05 * (d.exp() - d - 1) - obj, 0.0)
    n = ok.sum()
    if agg == llmcu.POLICY_TOKEN_MEAN:
        want = per.sum() / n
    elif agg == llmcu.POLICY_SEQUENCE_MEAN:
        want = (per.sum(1) / ok.sum(1).clamp(min=1)).mean()
    else:
        want = per.sum() / 100.0
    # the loss is a sum of terms of both signs: held to 1e-2 of their mean size (a ratio is off by about
    # 1e-3 of a log-probability of 8)
    size = (per.abs().sum() / n).item()
    assert abs(loss - want.item()) <= 1e-2 * size * (1 if agg != 2 else n.item() / 100), (loss, want.item())
    assert stats["tokens"] == n.item()
    cut = (ok & (r * A > r.clamp(0.8, 1.3) * A)).sum().item() / n.item()
    assert abs(stats["clipped"] - cut) < 1e-6
    c.check_grads(want)
    c.ctx.close()


def test_policy_equal_to_its_samples(llmcu, cuda_device):
    """With the step's own log-probabilities as the samples' every ratio is 1:
    the loss is minus the mean advantage, nothing clips even at a clip of 1e-3,
    and the KL to itself is 0."""
    c = Case(llmcu, batch=3, seq=40)
    lp = c.ctx.score(c.tok, c.tgt)
    adv = np.array([1.0, -2.0, 0.5], np.float32)
    loss, stats = c.ctx.policy_forward_backward(c.tok, c.tgt, lp, adv, llmcu.Policy(1e-3, 1e-3, 0.1), lp)
    ok = (c.tgt >= 0) & (c.tgt < c.cfg.vocab)
    want = -(ok * adv[:, None]).sum() / ok.sum()
    assert abs(loss - want) <= 1e-4 and stats["clipped"] == 0 and stats["kl"] <= 1e-7
    # and with no adapters' effect (B = 0) the preference loss against the base is log 2, its rewards 0
    c.ctx.close()
    c = Case(llmcu, batch=4, seq=40, lora_std=0)
    ref = c.ctx.score(c.tok, c.tgt, adapters=False)
    loss, rewards = c.ctx.preference_forward_backward(c.tok, c.tgt, llmcu.Preference(beta=0.1), ref)
    assert abs(loss - np.log(2)) <= 1e-4 and np.abs(rewards).max() <= 1e-3
    c.ctx.close()


def test_gradient_scale_does_not_matter(llmcu, cuda_device):
    """A loss a million times smaller or larger has the gradients scaled alike:
    the fp16 backward is carried at a scale of its own."""
    c = Case(llmcu, batch=4, seq=40, deterministic=True)
    old = c.ctx.score(c.tok, c.tgt)
    adv = np.array([1.0, -1.0, 0.5, 2.0], np.float32)
    grads = []
    for norm in (1.0, 2.0 ** 20, 2.0 ** -20):
        c.ctx.policy_forward_backward(c.tok, c.tgt, old, adv, llmcu.Policy(agg=llmcu.POLICY_CONSTANT, norm=norm))
        grads.append({k: v * norm for k, v in c.ctx.grads_dict().items()})
    for k in grads[0]:
        assert np.array_equal(grads[0][k], grads[1][k]) and np.array_equal(grads[0][k], grads[2][k]), k
        assert np.isfinite(grads[0][k]).all() and np.abs(grads[0][k]).max() > 0
    # zero advantages: zero gradients
    c.ctx.policy_forward_backward(c.tok, c.tgt, old, 0 * adv, llmcu.Policy())
    assert all((v == 0).all() for v in c.ctx.grads_dict().values())
    c.ctx.close()


@pytest.mark.parametrize("targets", ["attn", "all"])
def test_muon_matches_its_formula(llmcu, cuda_device, targets):
    """llmcu_muon on every adapter against the update written out (64 bits, singular values)."""
    from oracle import golden as G
    cfg = G.CFG_TINY
    model = llmcu.Model.tiny()
    mask = llmcu.TARGETS_ALL if targets == "all" else llmcu.TARGETS_ATTN
    ctx = llmcu.Context(model, llmcu.Lora(7, 14.0, mask), llmcu.Run(2, 32))
    ctx.init_base_synthetic(1)
    ctx.init_lora_synthetic(2)
    tok, tgt = G.make_tokens(cfg, 2, 32, 9)
    opt = llmcu.Muon(lr=0.02, momentum=0.9, weight_decay=0.1, match_rms=True)
    a, b, k = 3.4445, -4.7750, 2.0315
    mom = None
    for _ in range(2):
        ctx.forward_backward(tok, tgt)
        before, grads = ctx.lora_dict(), ctx.grads_dict()
        ctx.muon(opt)
        after = ctx.lora_dict()
        mom = {n: 0.9 * (mom[n] if mom else 0) + g.astype(np.float64) for n, g in grads.items()}
        for n, g in grads.items():
            U, s, Vh = np.linalg.svd(g + 0.9 * mom[n], full_matrices=False)
            v = s / (np.sqrt((s ** 2).sum()) + 1e-7)
            for _ in range(5):
                v = v * (a + b * v ** 2 + k * v ** 4)
            step = 0.02 * 0.2 * np.sqrt(max(g.shape)) * (U * v) @ Vh
            want = before[n] * (1 - 0.002) - step
            # the momentum is rounded to fp32, and five steps raise a small direction by at most 3.4445^5
            tol = 2.0 ** -24 * (4 * np.abs(want).max() + 4 * 485 * 0.02 * 0.2 * np.sqrt(max(g.shape)))
            assert np.abs(after[n] - want).max() <= tol, n
    # the momentum travels with the optimizer sidecar
    ctx.close()


def test_muon_resumes_from_the_sidecar(llmcu, cuda_device, tmp_path):
    c = Case(llmcu, batch=2, seq=32, deterministic=True)
    tgt = np.abs(c.tgt) % c.cfg.vocab
    opt = llmcu.Muon(lr=0.01)
    for _ in range(2):
        c.ctx.forward_backward(c.tok, tgt)
        c.ctx.muon(opt)
    c.ctx.save_lora(str(tmp_path), 2)
    c.ctx.save_adamw_state(str(tmp_path), 2)
    c.ctx.forward_backward(c.tok, tgt)
    c.ctx.muon(opt)
    want = c.ctx.lora_dict()
    c.ctx.load_lora(str(tmp_path), 2)
    c.ctx.load_adamw_state(str(tmp_path), 2)
    c.ctx.forward_backward(c.tok, tgt)
    c.ctx.muon(opt)
    got = c.ctx.lora_dict()
    assert all(np.array_equal(want[k], got[k]) for k in want)
    c.ctx.close()


def test_a_run_of_preference_steps(llmcu, cuda_device):
    """Reference scores, then preference steps with Muon and policy steps with
    AdamW; the same run twice (deterministic mode) gives the same bits."""
    ends = []
    for _ in range(2):
        c = Case(llmcu, batch=4, seq=40, seed=5, deterministic=True)
        start = c.ctx.lora_dict()
        ref = c.ctx.score(c.tok, c.tgt, adapters=False)
        cfg = llmcu.Preference(beta=0.1)
        for _ in range(3):
            c.ctx.preference_forward_backward(c.tok, c.tgt, cfg, ref)
            c.ctx.muon(llmcu.Muon(lr=1e-3))
        c.ctx.reset_optimizer()
        old = c.ctx.score(c.tok, c.tgt)
        for step in (1, 2):
            c.ctx.policy_forward_backward(c.tok, c.tgt, old, np.array([1, -1, 1, -1], np.float32),
                                          llmcu.Policy(kl_beta=0.02), ref)
            c.ctx.adamw(llmcu.AdamW(), step)
        ends.append(c.ctx.lora_dict())
        c.ctx.close()
        for k, v in ends[-1].items():
            assert np.isfinite(v).all() and not np.array_equal(v, start[k]), k
    assert all(np.array_equal(ends[0][k], ends[1][k]) for k in ends[0])


def test_int8_base_and_mlp_targets(llmcu, cuda_device):
    """The same losses over an INT8 base with adapters on every projection: the
    loss and the gradients follow their definition through the score (the policy
    equals its samples, so the loss is minus the mean advantage)."""
    from oracle import golden as G
    tok, tgt = G.make_tokens(G.CFG_TINY, 2, 64, 4)
    for in_gemm in (False, True):
        ctx = llmcu.Context(llmcu.Model.tiny(), llmcu.Lora(4, 8.0, llmcu.TARGETS_ALL if not in_gemm else 0x0F),
                            llmcu.Run(2, 64, base_dtype=llmcu.BASE_INT8, int8_in_gemm=in_gemm))
        ctx.init_base_synthetic(3)
        ctx.init_lora_synthetic(4)
        lp = ctx.score(tok, tgt)
        adv = np.array([2.0, 2.0], np.float32)
        loss, _ = ctx.policy_forward_backward(tok, tgt, lp, adv, llmcu.Policy())
        assert abs(loss + 2.0) <= 1e-4
        got = ctx.grads_dict()
        # -2 times the mean log-probability's gradient = 2 x the cross-entropy's over every position
        ctx2 = llmcu.Context(llmcu.Model.tiny(), ctx.lora, llmcu.Run(2, 64, base_dtype=llmcu.BASE_INT8,
                                                                    int8_in_gemm=in_gemm, loss_all_positions=True))
        ctx2.init_base_synthetic(3)
        ctx2.init_lora_synthetic(4)
        ctx2.forward_backward(tok, tgt)
        for k, want in ctx2.grads_dict().items():
            assert G.rel_l2(got[k], 2 * want) <= GRAD_RELL2, k
        ctx.close()
        ctx2.close()


def test_refusals_keep_the_context_usable(llmcu, cuda_device):
    c = Case(llmcu, batch=3, seq=40)
    old = np.zeros((3, 40), np.float32)
    adv = np.ones(3, np.float32)

    def refused(fn, *a):
        with pytest.raises(llmcu.LlmcuError) as e:
            fn(*a)
        assert e.value.status == 1

    refused(c.ctx.preference_forward_backward, c.tok, c.tgt, llmcu.Preference())  # three rows are no pairs
    refused(c.ctx.preference_forward_backward, c.tok[:2], c.tgt[:2], llmcu.Preference(beta=0.0))
    refused(c.ctx.policy_forward_backward, c.tok, c.tgt, old, adv, llmcu.Policy(clip_low=-1.0))
    refused(c.ctx.policy_forward_backward, c.tok, c.tgt, None, adv, llmcu.Policy())
    refused(c.ctx.muon, llmcu.Muon(ns_steps=0))
    refused(c.ctx.score, np.zeros((4, 40), np.int32), np.zeros((4, 40), np.int32))  # batch over max_batch
    bad = c.tok.copy()
    bad[0, 0] = c.cfg.vocab
    refused(c.ctx.score, bad, c.tgt)
    refused(c.ctx.policy_forward_backward, bad, c.tgt, old, adv, llmcu.Policy())
    with pytest.raises(ValueError):
        c.ctx.policy_forward_backward(c.tok, c.tgt, old[:, :7], adv, llmcu.Policy())
    with pytest.raises(ValueError):
        c.ctx.policy_forward_backward(c.tok, c.tgt, old, adv[:2], llmcu.Policy())
    lp = c.ctx.score(c.tok, c.tgt)
    assert np.isfinite(lp).all()
    loss, _ = c.ctx.policy_forward_backward(c.tok, c.tgt, lp, adv, llmcu.Policy())
    assert abs(loss + 1) < 1e-3
    c.ctx.close()


def test_llm_train_with_muon(cuda_device, tmp_path):
    """The driver's --optimizer muon runs, saves, and resumes to the same bits as the run in one piece."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = os.path.join(root, "llm.cu_b200", "llm_train")
    if not os.path.exists(exe):
        pytest.skip("llm_train not built")
    args = [exe, "--config", "tiny", "--synthetic", "--seq-len", "64", "--batch", "1", "--save-every", "2",
            "--log-every", "1", "--optimizer", "muon", "--lr", "1e-3", "--out", str(tmp_path)]
    one = subprocess.run(args + ["--steps", "3"], capture_output=True, text=True, timeout=120)
    assert one.returncode == 0, one.stderr
    losses = [line.split()[3] for line in one.stdout.splitlines() if line.startswith("step")]
    assert len(losses) == 3 and len(set(losses)) == 3
    two = subprocess.run(args + ["--steps", "3", "--resume", "2"], capture_output=True, text=True, timeout=120)
    assert two.returncode == 0, two.stderr
    assert [line.split()[3] for line in two.stdout.splitlines() if line.startswith("step")] == losses[2:]
    bad = subprocess.run([exe, "--optimizer", "sgd"], capture_output=True, text=True, timeout=30)
    assert bad.returncode == 1 and "unknown --optimizer" in bad.stderr
