"""Refusals of the preference-tuning operators, without a GPU: every case is
turned down by the host's checks before any device call."""
import dataclasses

import pytest

INVALID, UNSUPPORTED = 1, 8
P = 256 * 4096  # a stand-in for a device address: 256-byte aligned, never read


def refused(llmcu, status, fn, *args):
    with pytest.raises(llmcu.LlmcuError) as e:
        fn(*args)
    assert e.value.status == status, e.value


def lm(llmcu, backward, **kw):
    a = dict(x=P, E=P, targets=P, lse=P, dlogp=P, logp=P, dx=P, rows=4, hidden=64, vocab=512, ldx=64, lde=64, lddx=64,
             ws=P, nbytes=None)
    a.update(kw)
    if a["nbytes"] is None:
        a["nbytes"] = llmcu.lm_logprobs_workspace(4, 64, 512, backward)
    if backward:
        llmcu.lm_logprobs_bwd(a["x"], a["E"], a["targets"], a["lse"], a["dlogp"], a["dx"], a["rows"], a["hidden"],
                              a["vocab"], a["ldx"], a["lde"], a["lddx"], 1.0, a["ws"], a["nbytes"])
    else:
        llmcu.lm_logprobs(a["x"], a["E"], a["targets"], a["logp"], a["lse"], a["rows"], a["hidden"], a["vocab"],
                          a["ldx"], a["lde"], a["ws"], a["nbytes"])


@pytest.mark.parametrize("backward", [False, True])
def test_lm_logprobs_refusals(llmcu, backward):
    names = ["x", "E", "targets", "lse", "ws"] + (["dlogp", "dx"] if backward else ["logp"])
    for name in names:
        refused(llmcu, INVALID, lambda: lm(llmcu, backward, **{name: 0}))
    for kw in ({"rows": 0}, {"hidden": 0}, {"vocab": 0}, {"rows": -1}, {"ldx": 63}, {"lde": 56}, {"nbytes": 0}):
        refused(llmcu, INVALID, lambda: lm(llmcu, backward, **kw))
    size = llmcu.lm_logprobs_workspace(4, 64, 512, backward)
    refused(llmcu, INVALID, lambda: lm(llmcu, backward, nbytes=size - 1))
    refused(llmcu, UNSUPPORTED, lambda: lm(llmcu, backward, ws=P + 16))
    refused(llmcu, UNSUPPORTED, lambda: lm(llmcu, backward, targets=P + 2))
    # rows that the TMA cannot read
    refused(llmcu, UNSUPPORTED, lambda: lm(llmcu, backward, x=P + 8))
    refused(llmcu, UNSUPPORTED, lambda: lm(llmcu, backward, E=P + 2))
    refused(llmcu, UNSUPPORTED, lambda: lm(llmcu, backward, ldx=68))
    refused(llmcu, UNSUPPORTED, lambda: lm(llmcu, backward, lde=65))
    if backward:
        refused(llmcu, INVALID, lambda: lm(llmcu, backward, lddx=8))
        refused(llmcu, UNSUPPORTED, lambda: lm(llmcu, backward, dx=P + 1))


BIG = (1 << 31) - 1


def test_sizes_past_32_bits_are_refused(llmcu):
    """The largest ints a caller can pass are turned down, not wrapped around."""
    for kw in (dict(rows=BIG), dict(rows=(1 << 24) + 1), dict(hidden=BIG, ldx=BIG, lde=BIG, lddx=BIG),
               dict(vocab=BIG)):
        for backward in (False, True):
            refused(llmcu, UNSUPPORTED, lambda: lm(llmcu, backward, nbytes=1 << 60, **kw))
    assert llmcu.lm_logprobs_workspace(BIG, 64, 512) == 0 and llmcu.lm_logprobs_workspace(4, 64, BIG, True) == 0
    refused(llmcu, UNSUPPORTED, lambda: llmcu.preference_loss(llmcu.Preference(), P, 0, 0, 0, P, P, P, 1, BIG, BIG))
    refused(llmcu, UNSUPPORTED, lambda: llmcu.preference_loss(llmcu.Preference(), P, 0, 0, 0, P, P, P, BIG, 1, 1))
    refused(llmcu, UNSUPPORTED, lambda: llmcu.policy_loss(llmcu.Policy(), P, P, 0, P, 0, P, P, 1, BIG, BIG, P, 1 << 30))
    refused(llmcu, UNSUPPORTED, lambda: llmcu.policy_loss(llmcu.Policy(), P, P, 0, P, 0, P, P, 1 << 30, 1, 1, P,
                                                          1 << 40))
    refused(llmcu, UNSUPPORTED, lambda: llmcu.muon_update(llmcu.Muon(), P, P, P, 1, 16, BIG))
    refused(llmcu, UNSUPPORTED, lambda: llmcu.muon_update(llmcu.Muon(), P, P, P, 1, BIG, BIG))


def test_workspace_sizes(llmcu):
    assert llmcu.lm_logprobs_workspace(0, 64, 512) == 0 and llmcu.lm_logprobs_workspace(4, 64, -1, True) == 0
    assert llmcu.lm_logprobs_workspace(1, 2048, 151936) >= 4 + 8 * 1187
    # the backward holds one vocabulary chunk, never [rows, vocab]
    assert llmcu.lm_logprobs_workspace(4096, 2048, 151936, True) < 4096 * 151936 * 2 // 4
    assert llmcu.policy_loss_workspace(0, 4) == 0 and llmcu.policy_loss_workspace(7, 4) > 0


def test_preference_refusals(llmcu):
    good = llmcu.Preference(llmcu.PREF_SIGMOID, 0.1)

    def call(cfg=good, logp=P, pairs=2, seq=8, ld=8, dlogp=P):
        llmcu.preference_loss(cfg, logp, 0, 0, 0, P, P, dlogp, pairs, seq, ld)

    bad = [dict(kind=3), dict(kind=-1), dict(beta=0.0), dict(beta=-1.0), dict(beta=float("nan")),
           dict(beta=float("inf")), dict(label_smoothing=0.6), dict(label_smoothing=-0.1),
           dict(kind=llmcu.PREF_HINGE, label_smoothing=0.1), dict(kind=llmcu.PREF_SQUARED, margin=0.5),
           dict(margin=float("inf")), dict(mean_tokens=2)]
    for kw in bad:
        refused(llmcu, INVALID, call, dataclasses.replace(good, **kw))
    for kw in (dict(logp=0), dict(pairs=0), dict(pairs=-3), dict(seq=0), dict(ld=7)):
        refused(llmcu, INVALID, lambda: call(**kw))
    refused(llmcu, UNSUPPORTED, lambda: call(logp=P + 2))
    refused(llmcu, UNSUPPORTED, lambda: call(dlogp=P + 1))
    assert llmcu.lib().llmcu_preference_loss(None, P, 0, 0, 0, P, P, P, 1, 1, 1, 0) == INVALID


def test_policy_refusals(llmcu):
    good = llmcu.Policy()

    def call(cfg=good, logp=P, old=P, adv=P, stats=P, batch=2, seq=8, ld=8, ws=P, nbytes=1 << 20):
        llmcu.policy_loss(cfg, logp, old, 0, adv, 0, stats, P, batch, seq, ld, ws, nbytes)

    bad = [dict(clip_low=-0.1), dict(clip_high=float("nan")), dict(clip_high=float("inf")), dict(kl_beta=-1.0),
           dict(dual_clip=1.0), dict(dual_clip=0.5), dict(dual_clip=float("inf")), dict(agg=3), dict(agg=-1),
           dict(agg=llmcu.POLICY_CONSTANT, norm=0.0), dict(agg=llmcu.POLICY_CONSTANT, norm=float("nan")),
           dict(token_advantages=2)]
    for kw in bad:
        refused(llmcu, INVALID, call, dataclasses.replace(good, **kw))
    for kw in (dict(logp=0), dict(old=0), dict(adv=0), dict(stats=0), dict(ws=0), dict(batch=0), dict(seq=0),
               dict(ld=7), dict(nbytes=llmcu.policy_loss_workspace(2, 8) - 1)):
        refused(llmcu, INVALID, lambda: call(**kw))
    refused(llmcu, UNSUPPORTED, lambda: call(old=P + 1))
    refused(llmcu, UNSUPPORTED, lambda: call(ws=P + 128))
    # units of four tokens are counted in 31 bits
    refused(llmcu, UNSUPPORTED, lambda: call(batch=1 << 20, seq=1 << 14, ld=1 << 14, nbytes=1 << 30))


def test_muon_refusals(llmcu):
    good = llmcu.Muon()

    def call(cfg=good, w=P, g=P, m=P, count=2, rows=16, cols=64):
        llmcu.muon_update(cfg, w, g, m, count, rows, cols)

    for kw in (dict(lr=float("nan")), dict(momentum=float("inf")), dict(eps=0.0), dict(eps=-1.0), dict(ns_steps=0),
               dict(ns_steps=17), dict(nesterov=2), dict(match_rms=-1), dict(weight_decay=float("nan"))):
        refused(llmcu, INVALID, call, dataclasses.replace(good, **kw))
    for kw in (dict(w=0), dict(g=0), dict(m=0), dict(count=0), dict(rows=0), dict(cols=-2)):
        refused(llmcu, INVALID, lambda: call(**kw))
    refused(llmcu, UNSUPPORTED, lambda: call(w=P + 2))
    refused(llmcu, UNSUPPORTED, lambda: call(rows=17, cols=17))
