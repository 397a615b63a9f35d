"""The preference-tuning operators at the ends of their ranges: log-ratios whose
exponential leaves 32 bits, infinite log-probabilities of scored tokens, logits
past what the tensor cores resolve, and more than one vocabulary chunk."""
import ctypes as C
import math
import os
import subprocess
import time

import numpy as np
import pytest
import test_gpu_preference_ops as ops

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = ops.U
# one launch; the count and the main kernel (means), the main kernel and the sums (a constant divisor)
POLICY_CASES = [(8, 40, 43, 0), (8, 40, 43, 1), (8, 40, 43, 2), (40, 1500, 1501, 0), (40, 1500, 1501, 1),
                (40, 1500, 1501, 2)]


def policy_case(dev, B, S, ld, agg, seed):
    lp, old, rf, adv, mask = ops.policy_inputs(dev, B, S, ld, seed, True, empty=(1,))
    mask[:, ::7] = True  # the tokens that a test moves
    junk = mask & ~(lp.isfinite() & old.isfinite() & rf.isfinite() & (lp > -1e30) & (old > -1e30) & (rf > -1e30))
    return (*(torch.where(junk, -1.0, v) for v in (lp, old, rf)), adv, mask)


@pytest.mark.parametrize("B,S,ld,agg", POLICY_CASES)
def test_policy_without_kl_takes_any_reference(llmcu, cuda_device, B, S, ld, agg):
    """kl_beta 0: the reference reaches the KL statistic alone, whatever it holds."""
    lp, old, rf, adv, mask = policy_case(cuda_device, B, S, ld, agg, 3)
    cfg = llmcu.Policy(0.2, 0.28, 0.0, 3.0, agg, 0.7 * B * S, True)
    want = ops.run_policy(llmcu, cfg, lp, old, None, adv, mask, B, S, ld, cuda_device)
    assert want[0].isfinite().all()
    for far in (90.0, 200.0, 1000.0, float("inf"), float("-inf")):
        rf[:, 7] = lp[:, 7] + far
        rf[:, 14] = 0.0
        stats, d = ops.run_policy(llmcu, cfg, lp, old, rf, adv, mask, B, S, ld, cuda_device)
        assert torch.equal(d, want[1])
        assert torch.equal(stats[[0, 2, 3]], want[0][[0, 2, 3]])
        assert stats[1] > 1e30


@pytest.mark.parametrize("B,S,ld,agg", POLICY_CASES)
def test_policy_without_advantage_takes_any_ratio(llmcu, cuda_device, B, S, ld, agg):
    """An advantage of 0 makes the ratio's terms 0, however far it lies off."""
    lp, old, rf, adv, mask = policy_case(cuda_device, B, S, ld, agg, 4)
    for col, far in ((7, 90.0), (14, 99.0), (21, 300.0), (28, -300.0)):
        old[:, col] = lp[:, col] - far
        adv[:, col] = 0.0
    for dual in (0.0, 3.0):
        cfg = llmcu.Policy(0.2, 0.28, 0.04, dual, agg, 0.7 * B * S, True)
        ops.check_policy(llmcu, cfg, lp, old, rf, adv, mask, B, S, ld, cuda_device)
    adv.zero_()
    ops.check_policy(llmcu, cfg, lp, old, None, adv, mask, B, S, ld, cuda_device)
    old[:, 7] = float("nan")  # NaN stays to be seen
    stats, d = ops.run_policy(llmcu, cfg, lp, old, None, adv, mask, B, S, ld, cuda_device)
    assert stats[0].isnan() and d[mask[:, 7], 7].isnan().all()


@pytest.mark.parametrize("B,S,ld,agg", POLICY_CASES)
@pytest.mark.parametrize("dual", [0.0, 3.0])
def test_policy_exponentials_past_32_bits(llmcu, cuda_device, B, S, ld, agg, dual):
    """e^90 is past fp32; kl_beta or the advantage, and the weight, bring it back."""
    lp, old, rf, adv, mask = policy_case(cuda_device, B, S, ld, agg, 5)
    for row, col, far in ((0, 7, 90.0), (2, 14, 92.5), (3, 21, 88.5), (4, 7, 41.0), (5, 14, 39.0)):
        rf[row, col] = lp[row, col] + far
        old[row, col + 7] = lp[row, col + 7] - far
        adv[row, col + 7] = (1, -1)[row & 1] * 1e-4
    # both at once, one of them tiny
    rf[6, 7], old[6, 7] = lp[6, 7] + 91.0, lp[6, 7] - 1e-3
    rf[7, 7], old[7, 7], adv[7, 7] = lp[7, 7] + 1e-3, lp[7, 7] - 91.0, -1e-5
    cfg = llmcu.Policy(0.2, 0.28, 0.002, dual, agg, 0.7 * B * S, True)
    ops.check_policy(llmcu, cfg, lp, old, rf, adv, mask, B, S, ld, cuda_device)


@pytest.mark.parametrize("P,S", [(3, 5), (3, 9000)])
def test_preference_banned_tokens(llmcu, cuda_device, P, S):
    """A rejected sequence with a token of probability 0 is preferred without
    bounds: no loss, no gradient.  A chosen one loses without bounds."""
    dev = cuda_device
    lp = -torch.rand(2 * P, S, device=dev)
    lp[P, S // 2] = float("-inf")  # pair 0: rejected
    lp[1, S // 3] = float("-inf")  # pair 1: chosen
    cfg = llmcu.Preference(llmcu.PREF_SIGMOID, 0.5)
    loss, reward, d = ops.run_pref(llmcu, cfg, lp, None, None, None, P, S, S, dev)
    assert loss[0] == 0 and loss[1] == float("inf") and loss[2].isfinite()
    assert reward[P] == float("-inf") and reward[1] == float("-inf")
    assert (d[[0, P]] == 0).all()
    up = torch.tensor(1.0, device=dev) / P
    assert torch.equal(d[1], (-0.5 * up).expand(S)) and torch.equal(d[P + 1], (0.5 * up).expand(S))
    # smoothed labels hold a share of the other outcome, whose loss has no bound
    loss, _, d = ops.run_pref(llmcu, llmcu.Preference(llmcu.PREF_SIGMOID, 0.5, 0.1), lp, None, None, None, P, S, S, dev)
    assert (loss[:2] == float("inf")).all() and d.isfinite().all()
    loss, _, d = ops.run_pref(llmcu, llmcu.Preference(llmcu.PREF_HINGE, 0.5), lp, None, None, None, P, S, S, dev)
    assert loss[0] == 0 and loss[1] == float("inf") and (d[[0, P]] == 0).all()


@pytest.mark.parametrize("e", [1e-36, 1e-6, 0.01, 0.1, 0.3, 0.5])
def test_preference_smoothed_gradient_near_its_zero(llmcu, cuda_device, e):
    """Smoothed labels have a margin at which nothing pulls: the gradient keeps
    its digits on both sides of it.  One token a row and no reference, so that h
    is exact: off are t = h - h0 (rounded once, which moves e^t - 1 by at most
    2 (1 + |t|) half steps), expm1f (2) and ten products and sums."""
    dev = cuda_device
    e = float(torch.tensor(e))
    h0 = math.log((1 - e) / e)
    t = torch.logspace(-7, 2.5, 200, dtype=torch.float64)
    want_h = torch.cat([h0 - t, torch.tensor([h0]), h0 + t])
    P = len(want_h)
    cfg = llmcu.Preference(llmcu.PREF_SIGMOID, 0.5, e)
    # D = chosen - rejected in two fp32 parts, whose difference 64 bits hold
    D = want_h / 0.5
    high = D.float()
    lp = torch.cat([high, (high.double() - D).float()])[:, None].to(dev)
    D = (lp[:P, 0].double() - lp[P:, 0].double()).cpu()
    t = 0.5 * D - h0
    _, _, d = ops.run_pref(llmcu, cfg, lp, None, None, torch.ones(P, device=dev), P, 1, 1, dev)
    u, v = torch.expm1(-t.abs()), torch.exp(-t.abs())
    want = 0.5 * e * (1 - e) * torch.where(t > 0, -u / (1 - e + e * v), u / (e + (1 - e) * v))
    # the same as e - s(-h), as far as 64 bits tell them apart
    assert ((0.5 * (e - torch.sigmoid(-0.5 * D)) - want).abs() <= 2.0 ** -50).all()
    tol = (14 + 2 * t.abs().clamp(max=100)) * U * want.abs() + 2.0 ** -52
    ops.within(d[:P, 0].cpu(), want, tol)
    assert torch.equal(d[P:, 0], -d[:P, 0])


@pytest.mark.parametrize("M", [1, 5, 300])
@pytest.mark.parametrize("sign", [1, -1, 0])
def test_lm_logprobs_logits_past_their_rounding(llmcu, cuda_device, M, sign):
    """Logits of millions, whose roundings pass 100: the results are off by the
    logits' roundings and no more, a probability is never over 1 by more than a
    factor of two, and nothing is infinite."""
    dev, H, V = cuda_device, 2048, 700
    g = torch.Generator(device=dev).manual_seed(M)
    x = torch.randn(M, H, generator=g, device=dev) * 1000
    E = torch.randn(V, H, generator=g, device=dev) * 100
    if sign:
        x, E = x.abs(), sign * E.abs()
    x, E = x.half(), E.half()
    z = x.double() @ E.double().t()
    t = z.argmax(1).int()
    t[1::2] = torch.randint(0, V, (M // 2,), generator=g, device=dev, dtype=torch.int32)
    logp, lse = ops.lm_forward(llmcu, x, E, t)
    ref = torch.logsumexp(z, 1)
    tol = ops.logit_tol(x, E)
    assert tol.min() > 100
    lse_tol = tol + (64 + 4 * ref.abs() + 4 * z.abs().amax(1)) * U
    ops.within(lse, ref, lse_tol)
    ops.within(logp, z.gather(1, t.long()[:, None])[:, 0] - ref, lse_tol + tol + 2 * U * ref.abs())
    dlogp = torch.ones(M, device=dev)
    for slot in (t, (t + 1) % V):  # the likeliest column as the target and not
        dx = ops.lm_backward(llmcu, x, E, slot, lse, dlogp, 1.0)
        # (1 - p_t) E_t with 1 - p_t in [0, 1], and at most two columns near the top, each p at most 2
        assert dx.isfinite().all() and (dx.abs() <= 5 * E.abs().max()).all()


@pytest.mark.parametrize("M,H,V,chunks", [(4096, 64, 33000, 3), (9000, 8, 8000, 2), (4096, 64, 17000, 2),
                                          (100, 8, 1300000, 2)])
def test_lm_logprobs_backward_in_chunks(llmcu, cuda_device, M, H, V, chunks):
    """Several vocabulary chunks, the last one narrower and with fewer K slices
    than there are slabs; targets on both sides of every border.  The first shape
    has over 2^33 products, so that the rows with a gradient are gathered first."""
    dev = cuda_device
    x, E, t = ops.lm_case(dev, M, H, V, 7)
    # a chunk holds at most 2^26 probabilities in multiples of 1024 columns; its buffer shows in the workspace
    width = max(1024, (1 << 26) // M // 1024 * 1024)
    assert (V + width - 1) // width == chunks
    assert 2 * M * width < llmcu.lm_logprobs_workspace(M, H, V, True) < 2 * M * V + 2 * M * width
    border = [0, 1, V - 1, V - 2]
    for c in range(1, chunks):
        border += [c * width - 1, c * width, c * width + 1]
    t[10:10 + len(border)] = torch.tensor(border, dtype=torch.int32, device=dev)
    t[40::8], t[41] = -1, V
    live = (t >= 0) & (t < V)
    logp, lse = ops.lm_forward(llmcu, x, E, t)
    dlogp = torch.randn(M, generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    dlogp[43::8] = 0
    scale = 16.0
    dx = ops.lm_backward(llmcu, x, E, t, lse, dlogp, scale)
    assert torch.equal(dx, ops.lm_backward(llmcu, x, E, t, lse, dlogp, scale))
    Ed = E.double()
    for a in range(0, M, 1024):
        r = slice(a, min(a + 1024, M))
        z = x[r].double() @ Ed.t()
        picked = z.gather(1, t[r].long().clamp(0, V - 1)[:, None])[:, 0]
        p = torch.exp(z - lse[r].double()[:, None])
        w = torch.where(live[r], scale * dlogp[r].double(), 0.0)[:, None]
        Et = Ed[t[r].long().clamp(0, V - 1)]
        want = w * (Et - p @ Ed)
        # as for a single chunk, whose sums over K are in 32 bits too
        tol = ops.logit_tol(x[r], E)
        off = (tol + (8 + 4 * z.abs().amax(1) + 4 * lse[r].abs().double()) * U)[:, None]
        pt = torch.exp(picked - lse[r].double())[:, None]
        bound = w.abs() * ((p @ Ed.abs()) * (2.0 ** -11 + off + (V / 16 + 32) * 2 * U) +
                           2.0 ** -40 * Ed.abs().sum(0)[None] + Et.abs() * (pt * off + 4 * U))
        ops.within(dx[r], want, bound + want.abs() * (2.0 ** -11 + 8 * U) + 2.0 ** -25)
    assert (dx[~live] == 0).all() and (dx[dlogp == 0] == 0).all()
    assert llmcu.kernel_checks(ops.stream()) == 0


@pytest.mark.parametrize("M,H,V", [(4096, 64, 33000), (9000, 8, 8000)])
def test_lm_logprobs_backward_chunks_in_a_graph(llmcu, cuda_device, M, H, V):
    """The chunks' buffer is used again and again under programmatic launch: the same bits from a captured call."""
    dev = cuda_device
    x, E, t = ops.lm_case(dev, M, H, V, 8)
    t[5::9] = -1
    _, lse = ops.lm_forward(llmcu, x, E, t)
    dlogp = torch.randn(M, generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    want = ops.lm_backward(llmcu, x, E, t, lse, dlogp, 4.0)
    n = llmcu.lm_logprobs_workspace(M, H, V, True)
    ws, dx = torch.full((n,), 255, dtype=torch.uint8, device=dev), torch.zeros_like(want)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        llmcu.lm_logprobs_bwd(x.data_ptr(), E.data_ptr(), t.data_ptr(), lse.data_ptr(), dlogp.data_ptr(),
                              dx.data_ptr(), M, H, V, H, H, H, 4.0, ws.data_ptr(), n, ops.stream())
    for _ in range(3):
        dx.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, want)


# ------------------------------------------------------------- on a context
def context(llmcu, **run):
    from oracle import golden as G
    tok, tgt = G.make_tokens(G.CFG_TINY, 2, 40, 4)
    ctx = llmcu.Context(llmcu.Model.tiny(), llmcu.Lora(4, 8.0), llmcu.Run(2, 40, deterministic=True, **run))
    ctx.init_base_synthetic(3)
    ctx.init_lora_synthetic(4)
    return ctx, tok, tgt


def test_policy_step_without_kl_takes_any_reference(llmcu, cuda_device):
    """The default Policy() has kl_beta 0: a far reference leaves loss and adapter gradients as they are."""
    ctx, tok, tgt = context(llmcu)
    old = ctx.score(tok, tgt)
    adv = np.array([1.0, -0.5], np.float32)
    loss, stats = ctx.policy_forward_backward(tok, tgt, old, adv, llmcu.Policy())
    want = ctx.grads_dict()
    ref = old.copy()
    ref[0, 3], ref[1, 5] = old[0, 3] + 90, old[1, 5] + 200
    got = ctx.policy_forward_backward(tok, tgt, old, adv, llmcu.Policy(), ref)
    assert got[0] == loss and got[1]["clipped"] == stats["clipped"] and got[1]["kl"] > 1e30
    grads = ctx.grads_dict()
    assert all(np.array_equal(grads[k], want[k]) for k in want)
    ctx.close()


def busy(ctx, seconds):
    """Keeps the context's stream from its next work for so long, on the host."""
    nap = C.cast(C.CDLL(None).usleep, C.c_void_p)
    launch = C.CDLL("libcuda.so.1").cuLaunchHostFunc
    launch.argtypes = [C.c_void_p] * 3
    assert launch(ctx.stream(), nap, int(seconds * 1e6)) == 0


def test_score_and_steps_keep_their_deadline(llmcu, cuda_device):
    """A stream that does not move within the deadline ends the call in time,
    with nothing written behind its back; the context is usable again."""
    TIMEOUT = 6
    ctx, tok, tgt = context(llmcu)
    adv = np.ones(2, np.float32)
    old = ctx.score(tok, tgt)
    calls = [lambda: ctx.score(tok, tgt), lambda: ctx.forward_backward(tok, tgt),
             lambda: ctx.preference_forward_backward(tok, tgt, llmcu.Preference()),
             lambda: ctx.policy_forward_backward(tok, tgt, old, adv, llmcu.Policy())]
    for call in calls:
        call()  # whatever a first call loads is there
    for call in calls:
        ctx.dp_set_timeout_ms(200)
        busy(ctx, 1.5)
        t0 = time.monotonic()
        with pytest.raises(llmcu.LlmcuError) as e:
            call()
        assert e.value.status == TIMEOUT and time.monotonic() - t0 < 1.0
        torch.cuda.synchronize()
        ctx.dp_set_timeout_ms(60000)
        assert np.array_equal(ctx.score(tok, tgt), old)
    ctx.close()


def test_optimizers_do_not_take_each_others_moments(llmcu, cuda_device, tmp_path):
    """AdamW's moments and Muon's momentum share their memory and their file; each is refused to the other."""
    def refused(fn, *a):
        with pytest.raises(llmcu.LlmcuError) as e:
            fn(*a)
        assert e.value.status == 1 and "reset" in str(e.value)

    adamw, muon = llmcu.AdamW(), llmcu.Muon(lr=1e-3)
    ctx, tok, tgt = context(llmcu)
    ctx.forward_backward(tok, tgt)
    start = ctx.lora_dict()
    ctx.muon(muon)
    after = ctx.lora_dict()
    refused(ctx.adamw, adamw, 2)
    refused(ctx.train_step, tok, tgt, adamw, 2)
    assert all(np.array_equal(after[k], v) for k, v in ctx.lora_dict().items())
    ctx.muon(muon)  # it goes on
    ctx.save_adamw_state(str(tmp_path), 2)
    ctx.reset_optimizer()
    ctx.set_lora_dict(start)
    ctx.train_step(tok, tgt, adamw, 1)
    refused(ctx.muon, muon)
    ctx.train_step(tok, tgt, adamw, 2)
    ctx.save_adamw_state(str(tmp_path), 3)
    ctx.load_adamw_state(str(tmp_path), 2)  # Muon's
    refused(ctx.train_step, tok, tgt, adamw, 3)
    ctx.muon(muon)
    ctx.load_adamw_state(str(tmp_path), 3)  # AdamW's
    refused(ctx.muon, muon)
    ctx.train_step(tok, tgt, adamw, 4)
    ctx.reset_optimizer()
    ctx.muon(muon)
    # files without the optimizer's number: AdamW's second moment tells whose they are
    for step, mine, other in ((2, lambda: ctx.muon(muon), lambda: ctx.adamw(adamw, 3)),
                              (3, lambda: ctx.adamw(adamw, 4), lambda: ctx.muon(muon))):
        path = tmp_path / f"lora_step{step}_adamw.bin"
        raw = bytearray(path.read_bytes())
        raw[48:64] = bytes(16)
        path.write_bytes(raw)
        ctx.load_adamw_state(str(tmp_path), step)
        refused(other)
        mine()
    ctx.close()


def test_profile_counts_the_launches(llmcu, cuda_device):
    """Muon takes a launch for each cluster size, the losses one to two kernels beside the head's."""
    from oracle import golden as G
    m = llmcu.Model.tiny()
    tok, tgt = G.make_tokens(G.CFG_TINY, 2, 40, 4)
    old, adv = np.zeros((2, 40), np.float32), np.ones(2, np.float32)
    for targets in (llmcu.TARGETS_ATTN, llmcu.TARGETS_ALL):
        ctx = llmcu.Context(m, llmcu.Lora(4, 8.0, targets), llmcu.Run(2, 40))
        ctx.init_base_synthetic(3)
        ctx.init_lora_synthetic(4)
        ctx.profile_enable()

        def launches(kind, fn, *a):
            ctx.profile_read()
            fn(*a)
            return ctx.profile_read()[kind]["launches"]

        # 128 columns a CTA (few matrices), clusters of the next power of two up to eight
        sides = {m.hidden, m.n_heads * m.head_dim, m.n_kv_heads * m.head_dim}
        sides |= {m.ffn} if targets == llmcu.TARGETS_ALL else set()
        clusters = {min(8, 1 << (math.ceil(s / 128) - 1).bit_length()) for s in sides}
        ctx.forward_backward(tok, tgt)
        assert launches("adamw", ctx.muon, llmcu.Muon(lr=1e-3)) == len(clusters)
        ctx.reset_optimizer()
        assert launches("adamw", ctx.adamw, llmcu.AdamW(), 1) == 1
        # the cross-entropy finishes in two kernels; a loss in one of its own beside the
        # log-probabilities, the gradients' scale and the finishing kernel
        head = launches("lm_head", ctx.forward_backward, tok, tgt)
        assert launches("lm_head", ctx.preference_forward_backward, tok, tgt, llmcu.Preference()) == head + 2
        assert launches("lm_head", ctx.policy_forward_backward, tok, tgt, old, adv, llmcu.Policy()) == head + 2
        ctx.close()


@pytest.mark.parametrize("first,second", [("muon", "adamw"), ("adamw", "muon")])
def test_llm_train_does_not_resume_across_optimizers(cuda_device, tmp_path, first, second):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = os.path.join(root, "llm.cu_b200", "llm_train")
    args = [exe, "--config", "tiny", "--synthetic", "--seq-len", "32", "--batch", "1", "--save-every", "2",
            "--log-every", "1", "--lr", "1e-3", "--out", str(tmp_path)]
    one = subprocess.run(args + ["--steps", "2", "--optimizer", first], capture_output=True, text=True, timeout=120)
    assert one.returncode == 0, one.stderr
    two = subprocess.run(args + ["--steps", "3", "--resume", "2", "--optimizer", second], capture_output=True,
                         text=True, timeout=120)
    assert two.returncode != 0 and "reset" in two.stderr
    assert not os.path.exists(tmp_path / "lora_step3_layer0_wq_A.bin")
    same = subprocess.run(args + ["--steps", "3", "--resume", "2", "--optimizer", first], capture_output=True,
                          text=True, timeout=120)
    assert same.returncode == 0, same.stderr
