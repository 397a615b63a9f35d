"""The preference-tuning operators on the GPU against their formulas in 64 bits
on the same inputs.

Tolerances are elementwise and follow the roundings: u = 2^-24 is half a step of
fp32, fp16 rounds by at most 2^-11 relative.  A logit is a sum of exact products,
taken 16 at a time by the tensor cores: H / 16 additions to the accumulator and
up to 16 inside a step, each off by at most 2^-23 (a truncation) of the sum of
the absolute products."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def stream():
    return torch.cuda.current_stream().cuda_stream


def within(got, want, tol):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all() == torch.isfinite(want).all()
    over = (got - want).abs() - tol
    assert not (over > 0).any(), f"off by {(got - want).abs().max().item():.3g}, {over.max().item():.3g} too much"


# ------------------------------------------------------ token log-probabilities
def lm_case(dev, M, H, V, seed, pad=0, lean=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    E = (torch.randn(V, H + pad, generator=g, device=dev) * (0.9 / math.sqrt(H))).half()[:, :H]
    t = torch.randint(0, V, (M,), generator=g, device=dev, dtype=torch.int32)
    x = torch.randn(M, H, generator=g, device=dev)
    if lean:
        x += 14 * torch.rand(M, 1, generator=g, device=dev) * E[t.long()].float()
    buf = torch.zeros(M, H + pad, device=dev, dtype=torch.float16)
    buf[:, :H] = x.half()
    return buf[:, :H], E, t


def logit_tol(x, E):
    H = x.shape[1]
    return (H / 16 + 16) * 2 * U * (x.double().abs() @ E.double().abs().t()).amax(1)


def lm_forward(llmcu, x, E, t):
    M, H = x.shape
    V = E.shape[0]
    n = llmcu.lm_logprobs_workspace(M, H, V)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=x.device)  # NaN everywhere
    logp, lse = (torch.full((M,), float("nan"), device=x.device) for _ in range(2))
    llmcu.lm_logprobs(x.data_ptr(), E.data_ptr(), t.data_ptr(), logp.data_ptr(), lse.data_ptr(), M, H, V, x.stride(0),
                      E.stride(0), ws.data_ptr(), n, stream())
    return logp, lse


def lm_backward(llmcu, x, E, t, lse, dlogp, scale, pad=0):
    M, H = x.shape
    V = E.shape[0]
    n = llmcu.lm_logprobs_workspace(M, H, V, True)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=x.device)
    dx = torch.full((M, H + pad), 7.0, device=x.device, dtype=torch.float16)
    llmcu.lm_logprobs_bwd(x.data_ptr(), E.data_ptr(), t.data_ptr(), lse.data_ptr(), dlogp.data_ptr(), dx.data_ptr(), M,
                          H, V, x.stride(0), E.stride(0), H + pad, scale, ws.data_ptr(), n, stream())
    assert (dx[:, H:] == 7).all()
    return dx[:, :H]


SHAPES = [(1, 64, 128, 0), (1, 2048, 4096, 0), (2, 8, 1, 0), (3, 72, 127, 8), (128, 256, 129, 0), (129, 256, 4096, 0),
          (333, 200, 1000, 24), (257, 1024, 33000, 0), (40, 24, 20011, 0), (5, 13, 300, 3)]


@pytest.mark.parametrize("M,H,V,pad", SHAPES)
def test_lm_logprobs_forward_backward(llmcu, cuda_device, M, H, V, pad):
    x, E, t = lm_case(cuda_device, M, H, V, M + H + V, pad)
    if M > 2:
        t[1], t[2] = -1, V  # outside the vocabulary: scores nothing
    live = (t >= 0) & (t < V)
    logp, lse = lm_forward(llmcu, x, E, t)
    z = x.double() @ E.double().t()
    ref = torch.logsumexp(z, 1)
    picked = z.gather(1, t.long().clamp(0, V - 1)[:, None])[:, 0]
    tol = logit_tol(x, E)
    # the sum of exponentials: ex2's 2 ulp, the exponent's rounding and a few additions a slot
    lse_tol = tol + (64 + 4 * ref.abs() + 4 * z.abs().amax(1)) * U
    within(lse, ref, lse_tol)
    within(logp, torch.where(live, picked - ref, 0.0), lse_tol + tol + 2 * U * ref.abs())
    assert (logp[~live] == 0).all()

    g = torch.Generator(device=cuda_device).manual_seed(1)
    dlogp = torch.randn(M, generator=g, device=cuda_device)
    dlogp[~live] = float("nan")  # not used
    scale = 8.0
    dx = lm_backward(llmcu, x, E, t, lse, dlogp, scale, pad)
    p = torch.exp(z - lse.double()[:, None])
    Ed = E.double()
    w = torch.where(live, scale * dlogp.double(), 0.0)[:, None]
    want = w * (Ed[t.long().clamp(0, V - 1)] - p @ Ed)
    pt = torch.exp(picked - lse.double())[:, None]
    off = (tol + (8 + 4 * z.abs().amax(1) + 4 * lse.abs().double()) * U)[:, None]  # relative error of a probability
    bound = w.abs() * ((p @ Ed.abs()) * (2.0 ** -11 + off + (V / 16 + 32) * 2 * U) +
                       # probabilities under 2^-29 are fp16 subnormals (steps of 2^-24, times 2^-15)
                       2.0 ** -40 * Ed.abs().sum(0)[None] + Ed[t.long().clamp(0, V - 1)].abs() * (pt * off + 4 * U))
    bound = bound + want.abs() * 2.0 ** -11 + 2.0 ** -25 + 8 * U * want.abs()
    within(dx, want, bound)
    assert (dx[~live] == 0).all()
    # the same call gives the same bits
    assert torch.equal(dx, lm_backward(llmcu, x, E, t, lse, dlogp, scale, pad))
    assert all(torch.equal(a, b) for a, b in zip((logp, lse), lm_forward(llmcu, x, E, t)))
    assert llmcu.kernel_checks(stream()) == 0


def test_lm_logprobs_full_vocabulary(llmcu, cuda_device):
    """151,936 columns: several vocabulary chunks and K slices; a uniform row's probabilities lie at 2^-17."""
    M, H, V = 300, 2048, 151936
    x, E, t = lm_case(cuda_device, M, H, V, 3)
    x[7] = 0  # a uniform distribution
    t[11] = -7
    logp, lse = lm_forward(llmcu, x, E, t)
    assert abs(lse[7].item() - math.log(V)) < 4 * U * math.log(V) * 16
    z = x.double() @ E.double().t()
    ref = torch.logsumexp(z, 1)
    tol = logit_tol(x, E)
    within(lse, ref, tol + (64 + 4 * ref.abs() + 4 * z.abs().amax(1)) * U)
    dlogp = torch.linspace(-1, 1, M, device=cuda_device)
    dx = lm_backward(llmcu, x, E, t, lse, dlogp, 64.0)
    p = torch.exp(z - lse.double()[:, None])
    live = (t >= 0).double()[:, None]
    want = 64.0 * dlogp.double()[:, None] * live * (E.double()[t.long().clamp(0)] - p @ E.double())
    # roundings of many probabilities are independent: the whole is off by half a step or so of fp16
    assert ((dx.double() - want).norm() / want.norm()).item() < 2.0 ** -11
    assert (dx[11] == 0).all()


# from 2^33 products on the rows with a gradient are gathered first: the last
@pytest.mark.parametrize("M,H,V", [(1, 136, 5000), (2, 136, 5000), (257, 136, 5000), (1500, 136, 5000),
                                   (600, 511, 30000)])
@pytest.mark.parametrize("live", [0, 1, 0.03, 0.5])
def test_lm_logprobs_backward_rows_without_gradient(llmcu, cuda_device, M, H, V, live):
    """Rows whose upstream gradient is 0 or whose target scores nothing get zeros
    and leave the others' bits alone, from none of the rows to one and half of them."""
    x, E, t = lm_case(cuda_device, M, H, V, 6, pad=-H % 8)
    logp, lse = lm_forward(llmcu, x, E, t)
    g = torch.Generator(device=cuda_device).manual_seed(8)
    dlogp = torch.randn(M, generator=g, device=cuda_device)
    full = lm_backward(llmcu, x, E, t, lse, dlogp, 16.0)
    on = torch.rand(M, generator=g, device=cuda_device) < live if isinstance(live, float) else torch.zeros(
        M, dtype=torch.bool, device=cuda_device)
    if live == 1:
        on[M // 2] = True
    off = ~on
    half = torch.rand(M, generator=g, device=cuda_device) < 0.5
    t2 = torch.where(off & half, -100, t)
    d2 = torch.where(off & ~half, torch.zeros_like(dlogp), dlogp)
    d2 = torch.where(off & half, float("nan"), d2)
    got = lm_backward(llmcu, x, E, t2, lse, d2, 16.0)
    assert (got[off] == 0).all()
    x[off], lse[off] = float("nan"), float("nan")
    assert torch.equal(lm_backward(llmcu, x, E, t2, lse, d2, 16.0), got)
    # rows land in other tiles: the tensor cores' sums over K do not depend on the row
    assert torch.equal(got[on], full[on])
    assert llmcu.kernel_checks(stream()) == 0


def test_lm_logprobs_gradient_by_differences(llmcu, cuda_device):
    """Central differences of the forward along random directions.  A direction d
    of unit length moved by h = 1/8: the third derivative of logp along d is at
    most 2 |E_max|^3 <= 2 * 1.3^3, so the difference is off by h^2 / 6 of that;
    x is moved in fp16, and the step really taken is used."""
    M, H, V = 17, 128, 700
    x, E, t = lm_case(cuda_device, M, H, V, 9)
    logp, lse = lm_forward(llmcu, x, E, t)
    dx = lm_backward(llmcu, x, E, t, lse, torch.ones(M, device=cuda_device), 1.0).double()
    d = torch.randn(M, H, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(2))
    d = d / d.norm(dim=1, keepdim=True)
    h = 0.125
    xp, xm = (x.float() + h * d).half(), (x.float() - h * d).half()
    fp, fm = (lm_forward(llmcu, v, E, t)[0].double() for v in (xp, xm))
    # mean of the gradient along the step really taken
    slope = (dx * (xp.double() - xm.double())).sum(1)
    emax = E.double().norm(dim=1).amax().item()
    tol = 2 * h * (h * h / 6) * 2 * (emax * 1.1) ** 3 + 2 * logit_tol(x, E).max().item() * 2.2
    # the step is not quite symmetric: its middle lies up to an fp16 rounding from x
    mid = ((xp.double() + xm.double()) / 2 - x.double()).norm(dim=1).amax().item()
    tol += 2 * h * mid * emax ** 2 + 2 * h * 2.0 ** -11 * emax * 2
    within(fp - fm, slope, tol)


@pytest.mark.parametrize("M", [1, 2, 6])
def test_lm_logprobs_banned_and_extreme_logits(llmcu, cuda_device, M):
    """Rows of E that push their logits to -inf (banned ids) take no probability;
    logits of +-20000 neither overflow nor underflow the whole."""
    H, V = 64, 600
    x = torch.ones(M, H, device=cuda_device, dtype=torch.float16)
    E = (torch.randn(V, H, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(0)) * 0.1).half()
    E[::3] = float("-inf")
    E[128:256] = float("-inf")  # a whole slot of 128 columns
    t = torch.full((M,), 1, device=cuda_device, dtype=torch.int32)
    logp, lse = lm_forward(llmcu, x, E, t)
    z = x.double() @ E.double().t()
    within(lse, torch.logsumexp(z, 1), 1e-4)
    within(logp, torch.log_softmax(z, 1)[:, 1], 1e-4)
    E = torch.zeros(V, H, device=cuda_device, dtype=torch.float16)
    E[5], E[300] = 312.5, -312.5  # logits of +-20000
    logp, lse = lm_forward(llmcu, x, E, torch.tensor([5, 300, 0, 5, 300, 0], device=cuda_device, dtype=torch.int32)[:M])
    assert lse.tolist() == [20000.0] * M
    assert logp.tolist() == ([0.0, -40000.0, -20000.0] * 2)[:M]
    # a row whose every logit is -inf, and one with a NaN: no probability, no wrong number
    E[:] = float("-inf")
    logp, lse = lm_forward(llmcu, x, E, torch.zeros(M, device=cuda_device, dtype=torch.int32))
    assert (lse == float("-inf")).all() and logp.isnan().all()
    E.zero_()
    x[0, 3] = float("nan")
    logp, lse = lm_forward(llmcu, x, E, torch.zeros(M, device=cuda_device, dtype=torch.int32))
    assert lse[0].isnan() and logp[0].isnan()
    assert torch.allclose(lse[1:], torch.full_like(lse[1:], math.log(V)), rtol=1e-6)


# ------------------------------------------------------------- preference loss
def pref_inputs(dev, P, S, ld, seed, ref=True, empty=()):
    g = torch.Generator(device=dev).manual_seed(seed)
    rows = 2 * P
    lp = -torch.empty(rows, ld, device=dev).exponential_(0.8, generator=g)
    rf = lp + 0.3 * torch.randn(rows, ld, generator=g, device=dev)
    mask = torch.rand(rows, ld, generator=g, device=dev) < 0.7
    for e in empty:
        mask[e] = False
    # what is not scored must not be used, NaN and infinities included
    junk = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min], device=dev)
    pick = torch.randint(0, 4, (rows, ld), generator=g, device=dev)
    lp = torch.where(mask, lp, junk[pick])
    rf = torch.where(mask, rf, junk[pick.flip(0)])
    return lp, (rf if ref else None), mask


def pref_reference(llmcu, cfg, lp, rf, mask, dloss, P, S):
    m = mask[:, :S] if mask is not None else torch.ones(2 * P, S, dtype=torch.bool, device=lp.device)
    x = lp[:, :S].double().masked_fill(~m, 0).requires_grad_()
    z = x - (rf[:, :S].double().masked_fill(~m, 0) if rf is not None else 0)
    z = torch.where(m, z, 0.0)
    n = m.sum(1).clamp(min=1).double()
    R = z.sum(1) / (n if cfg.mean_tokens else 1)
    beta, e, margin = (float(v) for v in torch.tensor([cfg.beta, cfg.label_smoothing, cfg.margin]))
    D = R[:P] - R[P:]
    h = beta * D - margin
    F = torch.nn.functional
    if cfg.kind == llmcu.PREF_SIGMOID:
        loss = -(1 - e) * F.logsigmoid(h) - e * F.logsigmoid(-h)
    elif cfg.kind == llmcu.PREF_HINGE:
        loss = torch.relu(1 - h)
    else:
        loss = (D - 1 / (2 * beta)) ** 2
    up = dloss.double() if dloss is not None else torch.full((P,), 1 / P, dtype=torch.float64, device=lp.device)
    (loss * up).sum().backward()
    spread = (z.abs().sum(1) / (n if cfg.mean_tokens else 1)).detach()
    spread = spread[:P] + spread[P:]  # bounds the roundings of logp - ref
    return loss.detach(), (beta * R).detach(), x.grad, D.detach(), h.detach(), spread, beta


def run_pref(llmcu, cfg, lp, rf, mask, dloss, P, S, ld, dev):
    loss = torch.full((P,), float("nan"), device=dev)
    reward = torch.full((2 * P,), float("nan"), device=dev)
    dlogp = torch.full((2 * P, ld), 5.0, device=dev)
    ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    llmcu.preference_loss(cfg, lp.data_ptr(), ptr(rf), ptr(mask), ptr(dloss), loss.data_ptr(), reward.data_ptr(),
                          dlogp.data_ptr(), P, S, ld, stream())
    return loss, reward, dlogp


def check_pref(llmcu, cfg, lp, rf, mask, dloss, P, S, ld, dev):
    loss, reward, dlogp = run_pref(llmcu, cfg, lp, rf, mask, dloss, P, S, ld, dev)
    want, R, grad, D, h, spread, beta = pref_reference(llmcu, cfg, lp, rf, mask, dloss, P, S)
    dD = U * spread  # each logp - ref is rounded once
    if cfg.kind == llmcu.PREF_SQUARED:
        off = (D - 0.5 / beta).abs()
        tol = 2 * off * dD + 4 * U * want
        rel = dD / off.clamp(min=1e-30) + 8 * U
    else:
        tol = beta * dD + U * h.abs() + 8 * U * want.abs() + 2 * U * abs(cfg.margin)
        rel = 2 * (beta * dD + U * h.abs()) + 16 * U  # log s' and s' / s are at most 1 in size
    within(loss, want, tol)
    within(reward, R, torch.cat([beta * dD, beta * dD]) + 2 * U * R.abs())
    within(dlogp[:, :S], grad, torch.cat([rel, rel])[:, None] * grad.abs() + 1e-45)
    assert (dlogp[:, S:] == 5).all()
    m = mask[:, :S] if mask is not None else None
    if m is not None:
        assert (dlogp[:, :S][~m] == 0).all()
    again = run_pref(llmcu, cfg, lp, rf, mask, dloss, P, S, ld, dev)
    assert all(torch.equal(a, b) for a, b in zip((loss, reward, dlogp), again))


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("P,S,ld", [(1, 1, 1), (1, 3, 5), (3, 2, 2), (2, 511, 513), (5, 700, 700), (64, 130, 137),
                                    (1, 33000, 33000), (3, 8191, 8192), (700, 17, 17), (300, 4096, 4096)])
def test_preference_loss(llmcu, cuda_device, kind, P, S, ld):
    lp, rf, mask = pref_inputs(cuda_device, P, S, ld, P + S, empty=(0,) if P > 2 else ())
    if P > 4:
        mask[[3, P + 3]] = False  # both rows of a pair
    g = torch.Generator(device=cuda_device).manual_seed(4)
    dloss = torch.randn(P, generator=g, device=cuda_device)
    sig = kind == llmcu.PREF_SIGMOID
    sq = kind == llmcu.PREF_SQUARED
    for mean in (False, True):
        cfg = llmcu.Preference(kind, 0.2, 0.1 if sig else 0.0, 0.0 if sq else 0.25, mean)
        check_pref(llmcu, cfg, lp, rf, mask, None, P, S, ld, cuda_device)
        check_pref(llmcu, cfg, lp, rf, mask, dloss, P, S, ld, cuda_device)
    full = lp.nan_to_num(-1.0, -2.0, -3.0).clamp(-50, 0)
    check_pref(llmcu, llmcu.Preference(kind, 0.05, 0.0, 0.0, True), full, None, None, None, P, S, ld, cuda_device)


def test_preference_unaligned_bases(llmcu, cuda_device):
    """Bases one element past an aligned address: rows are then read element by element, with the same results."""
    P, S, ld = 4, 301, 303
    lp, rf, mask = pref_inputs(cuda_device, P, S, ld, 5)
    cfg = llmcu.Preference(llmcu.PREF_SIGMOID, 0.3)
    base = run_pref(llmcu, cfg, lp, rf, mask, None, P, S, ld, cuda_device)
    for which in range(4):
        bufs = []
        for i, v in enumerate((lp, rf, mask)):
            b = torch.empty(v.numel() + 1, dtype=v.dtype, device=cuda_device)
            s = b[1:] if which in (i, 3) else b[:-1]
            s.copy_(v.flatten())
            bufs.append(s)
        got = run_pref(llmcu, cfg, *bufs, None, P, S, ld, cuda_device)
        # the sums meet in another order only through their quads: 64-bit sums, so the fp32 results agree
        assert all(torch.allclose(a, b, rtol=4 * U, atol=0, equal_nan=True) for a, b in zip(base, got))


def test_preference_extreme_margins(llmcu, cuda_device):
    """Differences of +-1000: the loss is linear or 0 and its gradient beta or 0, never NaN."""
    lp = torch.tensor([[0.0], [-1000.0], [-1000.0], [0.0]], device=cuda_device)
    loss, reward, d = run_pref(llmcu, llmcu.Preference(llmcu.PREF_SIGMOID, 1.0), lp, None, None, None, 2, 1, 1,
                               cuda_device)
    assert loss.tolist() == [0.0, 1000.0] and reward.tolist() == [0.0, -1000.0, -1000.0, 0.0]
    assert d.flatten().tolist() == [0.0, -0.5, 0.0, 0.5]
    loss, _, d = run_pref(llmcu, llmcu.Preference(llmcu.PREF_HINGE, 1.0), lp, None, None, None, 2, 1, 1, cuda_device)
    assert loss.tolist() == [0.0, 1001.0] and d.flatten().tolist() == [0.0, -0.5, 0.0, 0.5]
    nan = torch.full((2, 1), float("nan"), device=cuda_device)
    for kind in range(3):
        loss, _, d = run_pref(llmcu, llmcu.Preference(kind, 1.0), nan, None, None, None, 1, 1, 1, cuda_device)
        assert loss.isnan().all() and d.isnan().all()


def test_preference_offsets_past_32_bits(llmcu, cuda_device):
    """Four rows 800 million elements apart: offsets pass 2^31."""
    P, S, ld = 2, 9, 800_000_001
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB of free device memory")
    lp, dl = (torch.empty(2 * P, ld, device=cuda_device) for _ in range(2))
    mask = torch.empty(2 * P, ld, dtype=torch.uint8, device=cuda_device)
    small = pref_inputs(cuda_device, P, S, S, 8, ref=False)
    lp[:, :S], mask[:, :S] = small[0], small[2].to(torch.uint8)
    cfg = llmcu.Preference(llmcu.PREF_SIGMOID, 0.3)
    loss, reward = torch.empty(P, device=cuda_device), torch.empty(2 * P, device=cuda_device)
    llmcu.preference_loss(cfg, lp.data_ptr(), 0, mask.data_ptr(), 0, loss.data_ptr(), reward.data_ptr(), dl.data_ptr(),
                          P, S, ld, stream())
    want = run_pref(llmcu, cfg, small[0], None, small[2], None, P, S, S, cuda_device)
    assert torch.allclose(loss, want[0], rtol=4 * U, atol=0)
    assert torch.allclose(dl[:, :S], want[2], rtol=4 * U, atol=0)


@pytest.mark.parametrize("agg", [0, 1, 2])
def test_policy_offsets_past_32_bits(llmcu, cuda_device, agg):
    """Three rows 1.1 billion elements apart (too many tokens for the one-launch kernel in the second half)."""
    B, ld = 3, 1_100_000_001
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GB of free device memory")
    lp, old, dl = (torch.empty(B, ld, device=cuda_device) for _ in range(3))
    mask = torch.empty(B, ld, dtype=torch.uint8, device=cuda_device)
    for S in (9, 12001):
        small = policy_inputs(cuda_device, B, S, S, 8, False)
        lp[:, :S], old[:, :S], mask[:, :S] = small[0], small[1], small[4].to(torch.uint8)
        cfg = llmcu.Policy(agg=agg, norm=50.0)
        n = llmcu.policy_loss_workspace(B, S)
        ws, stats = torch.empty(n, dtype=torch.uint8, device=cuda_device), torch.empty(4, device=cuda_device)
        llmcu.policy_loss(cfg, lp.data_ptr(), old.data_ptr(), 0, small[3].data_ptr(), mask.data_ptr(),
                          stats.data_ptr(), dl.data_ptr(), B, S, ld, ws.data_ptr(), n, stream())
        want = run_policy(llmcu, cfg, small[0], small[1], None, small[3], small[4], B, S, S, cuda_device)
        # the quads fall otherwise, and with them the order of the sums of up to four fp32 terms
        assert torch.equal(dl[:, :S], want[1])
        assert torch.allclose(stats, want[0], rtol=1e-5, atol=1e-6)


# ----------------------------------------------------------------- policy loss
def policy_inputs(dev, B, S, ld, seed, token_adv, empty=()):
    g = torch.Generator(device=dev).manual_seed(seed)
    lp = -torch.empty(B, ld, device=dev).exponential_(0.8, generator=g)
    old = lp + 0.25 * torch.randn(B, ld, generator=g, device=dev)
    rf = lp + torch.randn(B, ld, generator=g, device=dev) * torch.rand(B, ld, generator=g, device=dev) ** 6
    adv = torch.randn(*((B, ld) if token_adv else (B,)), generator=g, device=dev)
    mask = torch.rand(B, ld, generator=g, device=dev) < 0.6
    for e in empty:
        mask[e] = False
    junk = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min], device=dev)
    pick = torch.randint(0, 4, (B, ld), generator=g, device=dev)
    lp, old, rf = (torch.where(mask, v, junk[(pick + i) % 4]) for i, v in enumerate((lp, old, rf)))
    return lp, old, rf, adv, mask


def run_policy(llmcu, cfg, lp, old, rf, adv, mask, B, S, ld, dev, grads=True):
    n = llmcu.policy_loss_workspace(B, S)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=dev)
    stats = torch.full((4,), float("nan"), device=dev)
    d = torch.full((B, ld), 5.0, device=dev)
    ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    llmcu.policy_loss(cfg, lp.data_ptr(), old.data_ptr(), ptr(rf), adv.data_ptr(), ptr(mask), stats.data_ptr(),
                      d.data_ptr() if grads else 0, B, S, ld, ws.data_ptr(), n, stream())
    return stats, d


def check_policy(llmcu, cfg, lp, old, rf, adv, mask, B, S, ld, dev):
    stats, d = run_policy(llmcu, cfg, lp, old, rf, adv, mask, B, S, ld, dev)
    m = mask[:, :S] if mask is not None else torch.ones(B, S, dtype=torch.bool, device=dev)
    row, col = m.nonzero(as_tuple=True)
    x = lp[row, col].double().requires_grad_()
    o = old[row, col].double()
    A = (adv[row, col] if cfg.token_advantages else adv[row]).double()
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    beta, c = f32(cfg.kl_beta), f32(cfg.dual_clip)
    r = (x - o).exp()
    rc = r.clamp(1 - f32(cfg.clip_low), 1 + f32(cfg.clip_high))
    obj = torch.minimum(r * A, rc * A)
    cut = r * A > rc * A
    if c:
        cut = cut | ((A < 0) & (c * A > obj))
        obj = torch.where(A < 0, torch.maximum(obj, c * A), obj)
    dd = (rf[row, col].double() - x) if rf is not None else torch.zeros_like(x)
    kl = dd.expm1() - dd
    per = beta * kl - obj
    n, count = len(row), torch.bincount(row, minlength=B).double()
    if cfg.agg == llmcu.POLICY_TOKEN_MEAN:
        w = torch.full_like(A, 1 / max(n, 1))
    elif cfg.agg == llmcu.POLICY_SEQUENCE_MEAN:
        w = 1 / (count[row] * B)
    else:
        w = torch.full_like(A, 1 / f32(cfg.norm))
    loss = (per * w).sum()
    grad = torch.zeros(B, S, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(grad)
    if n:
        loss.backward()
        grad[row, col] = x.grad
        with torch.no_grad():
            delta, em1 = (x - o).abs(), dd.expm1().abs()
            # expf 2 ulp and its argument's rounding; expm1f 1 ulp and d's rounding; a few products
            t = w * ((r * A).abs() * (8 + delta) + beta * (8 * em1 + (dd.exp() * dd.abs()))) * U
            tol[row, col] = t + 8 * U * x.grad.abs()
    within(d[:, :S], grad, tol + 1e-45)
    assert (d[:, :S][~m] == 0).all() and (d[:, S:] == 5).all()
    with torch.no_grad():
        each = w * ((r * A).abs() * (8 + (x - o).abs()) + obj.abs() * 4 +
                    beta * (24 * kl + dd.expm1().abs() * dd.abs() + dd.abs() * (kl > 0.1))) * U
        mean = max(n, 1)
        kl_tol = ((24 * kl + dd.expm1().abs() * dd.abs() * 2 + dd.abs() * (kl > 0.1)) * U).sum() / mean
        want = [loss.detach(), kl.sum() / mean, cut.double().sum() / mean, float(n)]
        tols = [each.sum() + 4 * U * loss.abs(), kl_tol, 2 * U, 0.0]
    for got, v, t in zip(stats.double().tolist(), want, tols):
        assert abs(got - float(v)) <= float(t) + 1e-45, (stats.tolist(), [float(v) for v in want], float(t))
    again = run_policy(llmcu, cfg, lp, old, rf, adv, mask, B, S, ld, dev)
    assert torch.equal(stats, again[0]) and torch.equal(d, again[1])
    only = run_policy(llmcu, cfg, lp, old, rf, adv, mask, B, S, ld, dev, grads=False)
    assert torch.equal(stats, only[0]) and (only[1] == 5).all()


@pytest.mark.parametrize("agg", [0, 1, 2])
@pytest.mark.parametrize("B,S,ld", [(1, 1, 1), (1, 2, 3), (9, 1, 1), (5, 3, 3), (8, 512, 512), (7, 1025, 1031),
                                    (1, 20000, 20000), (2000, 5, 6), (33, 1023, 1023), (64, 4099, 4099)])
@pytest.mark.parametrize("token_adv", [False, True])
def test_policy_loss(llmcu, cuda_device, agg, B, S, ld, token_adv):
    v = policy_inputs(cuda_device, B, S, ld, B * S + agg, token_adv, empty=(1,) if B > 2 else ())
    lp, old, rf, adv, mask = v
    norm = 0.7 * B * S
    check_policy(llmcu, llmcu.Policy(0.2, 0.28, 0.04, 3.0, agg, norm, token_adv), lp, old, rf, adv, mask, B, S, ld,
                 cuda_device)
    check_policy(llmcu, llmcu.Policy(0.2, 0.2, 0.0, 0.0, agg, norm, token_adv), lp, old, None, adv, mask, B, S, ld,
                 cuda_device)
    full = [x.nan_to_num(-1.0, -2.0, -3.0).clamp(-3, 0) for x in (lp, old, rf)]
    check_policy(llmcu, llmcu.Policy(0.1, 0.3, 0.5, 2.0, agg, norm, token_adv), *full, adv, None, B, S, ld,
                 cuda_device)


def test_policy_all_masked(llmcu, cuda_device):
    lp, old, rf, adv, mask = policy_inputs(cuda_device, 3, 40, 40, 1, False)
    mask[:] = False
    for agg in range(3):
        stats, d = run_policy(llmcu, llmcu.Policy(agg=agg, kl_beta=0.1), lp, old, rf, adv, mask, 3, 40, 40, cuda_device)
        assert stats.tolist() == [0.0, 0.0, 0.0, 0.0] and (d == 0).all()


def test_policy_borders_and_wide_clips(llmcu, cuda_device):
    """The fp32 neighbours of each border fall on the side that 64 bits say; a
    lower clip of 1 or more never clips."""
    borders = [math.log(1 + float(torch.tensor(0.2))), math.log(1 - float(torch.tensor(0.2))), math.log(3.0)]
    vals = []
    for b in borders:
        v = torch.tensor(b, dtype=torch.float32)
        up, down = torch.nextafter(v, v + 1), torch.nextafter(v, v - 1)
        vals += [down, v, up]
    lp = torch.stack(vals).repeat(2).to(cuda_device)[None]
    adv = torch.tensor([1.0, -1.0], device=cuda_device).repeat_interleave(9)[None].contiguous()
    old = torch.zeros_like(lp)
    S = lp.shape[1]
    cfg = llmcu.Policy(0.2, 0.2, 0.0, 3.0, llmcu.POLICY_CONSTANT, 1.0, True)
    stats, d = run_policy(llmcu, cfg, lp, old, None, adv, None, 1, S, S, cuda_device)
    x, A = lp.double()[0], adv.double()[0]
    cut = ((A > 0) & (x > borders[0])) | ((A < 0) & (x < borders[1])) | ((A < 0) & (x > borders[2]))
    assert torch.equal(d[0] == 0, cut)
    assert abs(stats[2].item() * S - cut.sum().item()) < 1e-4
    wide = llmcu.Policy(1.5, 0.2, 0.0, 0.0, llmcu.POLICY_CONSTANT, 1.0, True)
    lp = torch.full((1, 8), -60.0, device=cuda_device)
    stats, d = run_policy(llmcu, wide, lp, torch.zeros_like(lp), None, -torch.ones_like(lp), None, 1, 8, 8, cuda_device)
    assert stats[2] == 0 and (d > 0).all()


def test_policy_small_kl_keeps_its_digits(llmcu, cuda_device):
    """e^d - d - 1 near 0, over eleven decades of d."""
    d = torch.logspace(-9, 2, 400, device=cuda_device).clamp(max=80.0)
    lp = torch.cat([-d, d])[:, None]
    zero = torch.zeros_like(lp)
    for i in (0, 50, 100, 200, 300, 340, 360, 399, 400, 500, 600, 700, 760):
        one = lp[i:i + 1].contiguous()
        stats, g = run_policy(llmcu, llmcu.Policy(kl_beta=1.0, agg=2), one, one, zero[:1], zero[0], None, 1, 1, 1,
                              cuda_device)
        x = -one.double().item()
        kl = math.expm1(x) - x if abs(x) > 1e-3 else x * x / 2 * (1 + x / 3 * (1 + x / 4 * (1 + x / 5)))
        assert abs(stats[1].item() - kl) <= (16 + 2 * abs(x)) * U * kl + 1e-38
        assert abs(g.item() + math.expm1(x)) <= (8 + 2 * abs(x)) * U * abs(math.expm1(x))


def test_loss_gradients_by_differences(llmcu, cuda_device):
    """Central differences of both losses along a random direction v, taken over
    the step really made in fp32.  Second derivatives along v are under 1 (beta^2
    |v|^2 / 4 and (|A| r + beta e^d) |v|^2), third ones too, so a step of h is
    off by at most h^3 / 3; each loss is off by 16 roundings of 1."""
    dev, B, S = cuda_device, 8, 24
    lp, old, rf, adv, mask = policy_inputs(dev, B, S, S, 3, True)
    v = torch.randn(B, S, device=dev, generator=torch.Generator(device=dev).manual_seed(1)) * mask
    v /= v.norm() * 4
    h = 2.0 ** -4
    up, down = (torch.where(mask, lp + s * h * v, lp) for s in (1, -1))
    step = torch.where(mask, up.double() - down.double(), 0.0)

    def pref(x, dloss=None):
        return run_pref(llmcu, llmcu.Preference(llmcu.PREF_SIGMOID, 0.3, 0.1), x, rf, mask, None, B // 2, S, S, dev)

    # wide clips: no token changes sides within the step
    cfg = llmcu.Policy(0.999, 50.0, 0.1, 0.0, llmcu.POLICY_TOKEN_MEAN, 1.0, True)

    def policy(x):
        return run_policy(llmcu, cfg, x, old, rf, adv, mask, B, S, S, dev)

    tol = h ** 3 / 3 + 2 * 16 * U
    diff = pref(up)[0].double().mean() - pref(down)[0].double().mean()
    assert abs(diff - (pref(lp)[2].double() * step).sum()) <= tol
    diff = policy(up)[0][0].double() - policy(down)[0][0].double()
    assert abs(diff - (policy(lp)[1].double() * step).sum()) <= tol


# ------------------------------------------------------------------ Muon update
NS = tuple(float(v) for v in torch.tensor([3.4445, -4.7750, 2.0315]))


def muon_reference(u, eps, steps):
    """Newton-Schulz on the singular values (64 bits)."""
    a, b, c = NS
    Um, s, Vh = torch.linalg.svd(u.double().cpu(), full_matrices=False)
    v = s / (s.square().sum(-1, keepdim=True).sqrt() + eps)
    for _ in range(steps):
        v = v * (a + b * v ** 2 + c * v ** 4)
    return ((Um * v[:, None, :]) @ Vh).to(u.device)


def muon_case(dev, n, rows, cols, seed, decades=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    k, m = min(rows, cols), max(rows, cols)
    mix = torch.randn(n, k, k, generator=g, device=dev) * torch.logspace(0, -decades, k, device=dev)
    v = [(torch.bmm(mix, torch.randn(n, k, m, generator=g, device=dev)) * s) for s in (1e-3, 5e-3)]
    v = [x if rows <= cols else x.transpose(1, 2) for x in v]
    w = torch.randn(n, rows, cols, generator=g, device=dev) * 0.02
    return w, v[0].contiguous(), v[1].contiguous()


@pytest.mark.parametrize("n,rows,cols", [(1, 1, 1), (2, 1, 7), (3, 5, 1), (2, 16, 16), (1, 8, 8), (2, 7, 9), (4, 16, 33),
                                         (3, 33, 16), (2, 9, 1000), (2, 1001, 11), (5, 16, 2048), (5, 2048, 16),
                                         (1, 16, 13000), (1, 12345, 16), (1, 3, 30001), (130, 16, 256), (700, 4, 40),
                                         (40, 6144, 16), (40, 16, 6144)])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_update(llmcu, cuda_device, n, rows, cols, nesterov):
    w, g, mom = muon_case(cuda_device, n, rows, cols, n + rows + cols)
    if n > 2:
        g[1], mom[1] = 0, 0  # nothing to orthogonalise
    cfg = llmcu.Muon(lr=1.0, momentum=0.95, weight_decay=0.25, nesterov=nesterov, match_rms=not nesterov)
    w0, m0 = w.clone(), mom.clone()
    llmcu.muon_update(cfg, w.data_ptr(), g.data_ptr(), mom.data_ptr(), n, rows, cols, stream())
    mu = float(torch.tensor(0.95))
    want = mu * m0.double() + g.double()
    within(mom, want, 2 * U * (want.abs() + (mu * m0.double()).abs()))
    # the update from the momentum as it was stored, rounded once like the kernel's
    u = (mu * mom.double() + g.double()).float() if nesterov else mom
    X = muon_reference(u, cfg.eps, 5)
    s = 0.2 * math.sqrt(max(rows, cols)) if cfg.match_rms else math.sqrt(max(1.0, rows / cols))
    # X in 64 bits, rounded to fp32; s, the product and the sum in fp32
    want = 0.75 * w0.double() - s * X
    within(w, want, U * (4 * s * X.abs() + 2 * want.abs() + 2 * w0.double().abs()) + 1e-12 * s * X.abs().amax())
    if n > 2:
        assert torch.equal(w[1], 0.75 * w0[1])
    w2, m2 = w0.clone(), m0.clone()
    llmcu.muon_update(cfg, w2.data_ptr(), g.data_ptr(), m2.data_ptr(), n, rows, cols, stream())
    assert torch.equal(w, w2) and torch.equal(mom, m2)


@pytest.mark.parametrize("steps", [1, 2, 16])
@pytest.mark.parametrize("rows,cols", [(16, 100), (100, 6)])
def test_muon_steps_and_spectrum(llmcu, cuda_device, rows, cols, steps):
    """Directions four orders of magnitude apart keep their digits at any number of steps."""
    w, g, mom = muon_case(cuda_device, 3, rows, cols, 5, decades=4.0)
    w.zero_()
    mom.zero_()
    cfg = llmcu.Muon(lr=1.0, momentum=0.0, weight_decay=0.0, nesterov=False, ns_steps=steps)
    llmcu.muon_update(cfg, w.data_ptr(), g.data_ptr(), mom.data_ptr(), 3, rows, cols, stream())
    assert torch.equal(mom, g)
    X = muon_reference(g, cfg.eps, steps) * -math.sqrt(max(1.0, rows / cols))
    # 64-bit roundings, raised by at most 3.4445 a step (the small directions) until they saturate near 1
    amp = min(3.4445 ** steps, 1e5)
    within(w, X, 4 * U * X.abs() + 1e3 * 2.0 ** -53 * amp ** 2)


def test_muon_unaligned_base(llmcu, cuda_device):
    n, rows, cols = 3, 16, 260
    w, g, mom = muon_case(cuda_device, n, rows, cols, 2)
    cfg = llmcu.Muon()
    shifted = []
    for v in (w, g, mom):
        b = torch.empty(v.numel() + 1, device=cuda_device)
        b[1:] = v.flatten()
        shifted.append(b[1:])
    llmcu.muon_update(cfg, w.data_ptr(), g.data_ptr(), mom.data_ptr(), n, rows, cols, stream())
    llmcu.muon_update(cfg, *(v.data_ptr() for v in shifted), n, rows, cols, stream())
    assert torch.equal(shifted[0], w.flatten()) and torch.equal(shifted[2], mom.flatten())


# ------------------------------------------------- streams, graphs, the chain
def test_operators_as_one_chain_in_a_graph(llmcu, cuda_device):
    """hidden states -> log-probabilities -> losses -> gradient -> Muon update, on
    a side stream, captured and replayed with new inputs in place; two graphs with
    workspaces of their own replay at the same time."""
    dev = cuda_device
    P, S, H, V, r = 3, 50, 256, 4096, 16
    M = 2 * P * S

    def build(seed):
        x, E, t = lm_case(dev, M, H, V, seed)
        b = {"x": x.clone(), "E": E, "t": t, "mask": torch.rand(2 * P, S, device=dev) < 0.7}
        b["ref"] = -torch.rand(2 * P, S, device=dev) * 3
        b["old"] = -torch.rand(2 * P, S, device=dev) * 3
        b["adv"] = torch.randn(2 * P, device=dev)
        for k in ("logp", "lse", "d1", "d2"):
            b[k] = torch.empty(2 * P, S, device=dev)
        b["dx"] = torch.empty(M, H, device=dev, dtype=torch.float16)
        b["loss"], b["stats"] = torch.empty(P, device=dev), torch.empty(4, device=dev)
        b["w"], b["mom"] = torch.zeros(r, H, device=dev), torch.zeros(r, H, device=dev)
        b["g"] = torch.empty(r, H, device=dev)
        b["B"] = torch.randn(r, M, device=dev, dtype=torch.float16)
        sizes = [llmcu.lm_logprobs_workspace(M, H, V), llmcu.lm_logprobs_workspace(M, H, V, True),
                 llmcu.policy_loss_workspace(2 * P, S)]
        b["ws"] = [torch.empty(n, dtype=torch.uint8, device=dev) for n in sizes]
        return b

    def chain(b):
        st = stream()
        w1, w2, w3 = b["ws"]
        p = {k: v.data_ptr() for k, v in b.items() if k != "ws"}
        llmcu.lm_logprobs(p["x"], p["E"], p["t"], p["logp"], p["lse"], M, H, V, H, H, w1.data_ptr(), w1.numel(), st)
        llmcu.preference_loss(llmcu.Preference(beta=0.2), p["logp"], p["ref"], p["mask"], 0, p["loss"], 0, p["d1"], P, S,
                              S, st)
        llmcu.policy_loss(llmcu.Policy(kl_beta=0.05), p["logp"], p["old"], p["ref"], p["adv"], p["mask"], p["stats"],
                          p["d2"], 2 * P, S, S, w3.data_ptr(), w3.numel(), st)
        b["d1"].add_(b["d2"])
        llmcu.lm_logprobs_bwd(p["x"], p["E"], p["t"], p["lse"], p["d1"], p["dx"], M, H, V, H, H, H, 64.0, w2.data_ptr(),
                              w2.numel(), st)
        torch.mm(b["B"].float(), b["dx"].float(), out=b["g"])
        llmcu.muon_update(llmcu.Muon(), p["w"], p["g"], p["mom"], 1, r, H, st)

    keep = ("logp", "lse", "loss", "stats", "d1", "dx", "w", "mom")
    sets = [build(1), build(2)]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    eager, graphs = [], []
    for b, s in zip(sets, side):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            chain(b)
            s.synchronize()
            eager.append({k: b[k].clone() for k in keep})
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                chain(b)
            graphs.append(g)
    for rep in range(3):
        for b in sets:
            for k in keep:
                b[k].zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b, want in zip(sets, eager):
            for k in keep:
                assert torch.equal(b[k], want[k]), k
    assert eager[0]["w"].abs().sum() > 0 and eager[0]["dx"].abs().sum() > 0
    # new inputs in place
    sets[0]["x"].copy_(sets[1]["x"])
    sets[0]["E"].copy_(sets[1]["E"])
    sets[0]["t"].copy_(sets[1]["t"])
    torch.cuda.synchronize()
    with torch.cuda.stream(side[0]):
        graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(sets[0]["logp"], eager[1]["logp"])
    assert llmcu.kernel_checks(stream()) == 0
