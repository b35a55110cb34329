"""The serving operators inside the engine (whisper_full and whisper_decode): draws at a temperature on the device
(wmi_set_device_draws) and chunked self-attention for prompts (wmi_set_prompt_attention)."""
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from handy_amd.synth import synth_pcm    # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wr():
    from handy_amd import whisper_rs
    return whisper_rs


def _params(wr, best_of, temperature=0.8, inc=0.0):
    fp = wr.FullParams(wr.SamplingStrategy.Greedy(best_of))
    fp.set_temperature(temperature); fp.set_temperature_inc(inc); fp.set_language("en")
    return fp


def test_device_draws_of_one_token_are_the_most_probable_one(wr, model_path):
    """top_k = 1, min_p = 1 and a tiny top_p leave the most probable token only: the three give one transcript, whatever the random
    numbers -- for one decoder and for the best of four, alone and in a batch, with replayed passes and with plain launches."""
    ctx = wr.WhisperContext(model_path("micro.en", decisive=1.0))
    pcms = [synth_pcm(700 + i, 6 * 16000) for i in range(5)]
    st = ctx.create_batch_state(len(pcms), 4, 4)
    outs = []
    for best_of, kw in ((1, dict(top_k=1)), (1, dict(min_p=1.0)), (1, dict(top_p=1e-6)), (4, dict(top_k=1)), (4, dict(top_k=1, top_p=0.5, min_p=0.5))):
        st.set_device_draws(True, **kw)
        for graphs in (True, False):
            st.set_pass_graphs(graphs)
            st.full_batch(_params(wr, best_of), pcms)
            outs.append([st.batch_tokens(u) for u in range(len(pcms))])
    assert all(len(t) > 0 for t in outs[0])
    for o in outs[1:]:
        assert o == outs[0]
    one = ctx.create_state()
    one.set_device_draws(True, top_k=1)
    for pcm, ref in zip(pcms, outs[0]):
        one.full(_params(wr, 1), pcm)
        assert one.batch_tokens(0) == ref
    one.free(); st.free(); ctx.free()


def test_device_draws_repeat_and_differ(wr, model_path):
    """Without filters: every run draws the same tokens, other ones than the most probable, and the best of four is on some clip not
    the lone decoder's; log-probabilities are logarithms of probabilities; the fallback ladder runs to its end as with the host's draws."""
    ctx = wr.WhisperContext(model_path("micro.en", decisive=1.0))
    pcms = [synth_pcm(500 + i, 6 * 16000) for i in range(6)]
    out = {}
    for k in (1, 4):
        st = ctx.create_batch_state(len(pcms), 4, 4)
        st.set_device_draws(True)
        fp = _params(wr, k)
        st.full_batch(fp, pcms)
        out[k] = [st.batch_tokens(u) for u in range(len(pcms))]
        assert all(p <= 0.0 and np.isfinite(p) for u in range(len(pcms)) for s in st.batch_segments(u) for p in s.plog)
        st.full_batch(fp, pcms)
        assert [st.batch_tokens(u) for u in range(len(pcms))] == out[k]
        st.set_device_draws(True, top_k=1)
        st.full_batch(fp, pcms)
        assert [st.batch_tokens(u) for u in range(len(pcms))] != out[k]
        st.set_device_draws(False)                       # and the host's draws are what they were
        st.full_batch(fp, pcms)
        host = [st.batch_tokens(u) for u in range(len(pcms))]
        fresh = ctx.create_batch_state(len(pcms), 4, 4)
        fresh.full_batch(fp, pcms)
        assert [fresh.batch_tokens(u) for u in range(len(pcms))] == host
        fresh.free(); st.free()
    assert sum(a != b for a, b in zip(out[1], out[4])) >= 1
    fp = wr.FullParams(wr.SamplingStrategy.Greedy(2))    # default temperatures: random weights walk the whole ladder
    st = ctx.create_batch_state(len(pcms), 2, 2)
    st.full_batch(fp, pcms)
    fb = [st.batch_n_fallbacks(u) for u in range(len(pcms))]
    st.set_device_draws(True, top_p=0.9)
    st.full_batch(fp, pcms)
    assert [st.batch_n_fallbacks(u) for u in range(len(pcms))] == fb and sum(fb) > 0
    for kw in (dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=float("nan")), dict(top_p=float("nan"))):
        with pytest.raises(wr.WhisperError):
            st.set_device_draws(True, **kw)
    st.free(); ctx.free()


def test_device_draws_come_after_the_filter(wr, model_path):
    """What the caller's logits filter removes is never drawn: it leaves one token, then two, and the draws are those."""
    ctx = wr.WhisperContext(model_path("micro.en", decisive=1.0))
    pcm = synth_pcm(900, 6 * 16000)
    seen = set()
    for keep in ([1234], [1234, 777]):
        def only(tokens, logits, keep=keep):
            kept = logits[keep].copy()
            logits[:] = -np.inf
            logits[keep] = kept
        fp = _params(wr, 3)
        fp.set_no_timestamps(True); fp.set_max_tokens(12); fp.set_filter_logits_callback(only)
        st = ctx.create_batch_state(1, 4, 1)
        st.set_device_draws(True)
        st.full_batch(fp, [pcm])
        toks = st.batch_tokens(0)
        assert len(toks) > 0 and set(toks) <= set(keep), toks
        seen |= set(toks)
        st.free()
    assert seen == {1234, 777}
    ctx.free()


def test_window_memo_forgets_when_the_draws_change(wr, model_path):
    """A window remembered under one way of drawing is not taken over under another."""
    ctx = wr.WhisperContext(model_path("micro.en"))
    full = synth_pcm(41, 77 * 16000)
    full[8 * 16000:] *= 0.4
    fp = wr.FullParams(wr.SamplingStrategy.Greedy(2)); fp.set_language("en")
    settings = [(False, {}), (True, {}), (True, dict(top_k=5)), (True, dict(top_p=0.7)), (True, dict(min_p=0.2))]
    memo = ctx.create_batch_state(1, 2, 1)
    memo.set_window_cache(32)
    for on, kw in settings + settings[:2]:
        memo.set_device_draws(on, **kw)
        memo.full_batch(fp, [full])
        plain = ctx.create_batch_state(1, 2, 1)
        plain.set_device_draws(on, **kw)
        plain.full_batch(fp, [full])
        assert memo.batch_tokens(0) == plain.batch_tokens(0), (on, kw)
        plain.free()
    assert memo.window_cache_stats()["hits"] > 0         # the last two settings came back
    memo.free(); ctx.free()


@pytest.mark.parametrize("arch", ["mini", "mini512", "mini768"])
def test_prompt_attention_logits_match_the_oracle(wr, oracle, model_path, arch):
    """whisper_decode of 1 .. 250 tokens at once, and of chunks behind a cached prefix, with the chunked attention. The bound is the one
    the single-row kernel is held to (1e-2: a dozen fp16 roundings a layer; this adds one, of the probabilities)."""
    path = model_path(arch)
    om = oracle.OracleModel(path); ost = oracle.OracleState(om)
    ctx = wr.WhisperContext(path); st = ctx.create_state()
    pcm = synth_pcm(5, 10 * 16000)
    ost.pcm_to_mel(pcm); st.pcm_to_mel(pcm)
    ost.encode(0); st.encode(0)
    rng = np.random.default_rng(17)
    toks = [om.special("sot")] + [int(t) for t in rng.integers(0, 50000, size=249)]
    lref = ost.decode(toks, 0, 0, logits_all=True)
    base, base_one = st.decode_logits_all(toks, 0), st.decode_logits_all(toks[:1], 0)
    st.set_prompt_attention(True)
    for n in (250, 1, 2, 16, 17, 64, 65, 130):
        got = st.decode_logits_all(toks[:n], 0)
        assert float(np.abs(got - lref[:n]).max()) <= 1e-2, n
        if n == 1:
            assert np.array_equal(got, base_one)         # one token: the single-row kernel as ever
    st.decode(toks[:100], 0)                              # a cached prefix, then chunks of several sizes behind it
    at = 100
    for n in (1, 7, 40, 102):
        got = st.decode_logits_all(toks[at:at + n], at)
        assert float(np.abs(got - lref[at:at + n]).max()) <= 1e-2, (at, n)
        at += n
    nxt = st.decode([1234], 250)
    assert float(np.abs(nxt - ost.decode([1234], 250, 0)[0]).max()) <= 1e-2
    st.set_prompt_attention(False)
    assert np.array_equal(st.decode_logits_all(toks, 0), base)
    st.free(); ctx.free(); ost.close(); om.close()


def test_prompt_attention_keeps_the_transcripts(wr, model_path):
    """Prompts of different lengths in one batch (text context carried between windows, prompt tokens of the call): the tokens of the
    single-row kernel, with replayed passes and plain launches, alone and in a batch, and without prompt tokens. (Against the oracle these
    "varied" weights part by the encoder's rounding, with the single-row kernel at the same steps: see
    test_greedy_streams_on_varied_weights. The next test has the oracle's tokens.)"""
    ctx = wr.WhisperContext(model_path("micro", decisive=4.0, style="varied"))
    pcms = [synth_pcm(600 + i, int(s * 16000)) for i, s in enumerate((12.0, 65.0, 31.0, 3.0))]
    prompt = [int(t) for t in np.random.default_rng(3).integers(100, 40000, size=150)]
    for with_prompt in (True, False):
        fp = wr.FullParams(wr.SamplingStrategy.Greedy(1)); fp.set_temperature_inc(0.0); fp.set_language("en")
        if with_prompt:
            fp.set_tokens(prompt)
        plain = ctx.create_batch_state(len(pcms), 1, 4)
        plain.full_batch(fp, pcms)
        ref = [plain.batch_tokens(u) for u in range(len(pcms))]
        st = ctx.create_batch_state(len(pcms), 1, 4)
        st.set_prompt_attention(True)
        for graphs in (True, True, False):
            st.set_pass_graphs(graphs)
            st.full_batch(fp, pcms)
            assert [st.batch_tokens(u) for u in range(len(pcms))] == ref
        one = ctx.create_state()
        one.set_prompt_attention(True)
        for pcm, r in zip(pcms, ref):
            one.full(fp, pcm)
            assert one.batch_tokens(0) == r and len(r) > 0
        one.free(); st.free(); plain.free()
    ctx.free()


@pytest.mark.parametrize("arch", ["micro.en", "micro-v3"])
def test_prompt_attention_transcripts_match_the_oracle(wr, oracle, model_path, arch):
    """Greedy on plain weights with decisive margins, whose tokens are the oracle's with the single-row kernel: they are with the chunked
    one, over several windows with carried text, on one state and in a batch."""
    path = model_path(arch, decisive=4.0)
    om = oracle.OracleModel(path)
    ctx = wr.WhisperContext(path)
    fp = wr.FullParams(wr.SamplingStrategy.Greedy(1)); fp.set_temperature_inc(0.0); fp.set_language("en"); fp.set_no_context(False)
    op = oracle.default_params(0); op.temperature_inc = 0.0; op.best_of = 1; op.language = b"en"; op.no_context = 0
    pcms = [synth_pcm(10 + i, int(16000 * s)) for i, s in enumerate((30.0, 47.0, 4.0, 61.0))]
    st = ctx.create_batch_state(len(pcms), 1, 4)
    st.set_prompt_attention(True)
    st.full_batch(fp, pcms)
    for u, pcm in enumerate(pcms):
        o = oracle.OracleState(om)
        ref = [t for s in o.full(op, pcm) for t in s["tokens"]]
        one = ctx.create_state()
        one.set_prompt_attention(True)
        one.full(fp, pcm)
        assert st.batch_tokens(u) == ref and one.batch_tokens(0) == ref and len(ref) > 0
        one.free(); o.close()
    st.free(); ctx.free(); om.close()


def test_device_draws_where_nothing_is_left_take_the_rows_own_token(wr, model_path):
    """A caller's filter that leaves nothing on the prompt row of the second window: every one of the best-of-three decoders starts with what that
    row selects (id 0), none with the token it had selected last in the window before."""
    ctx = wr.WhisperContext(model_path("micro.en", decisive=1.0))
    prompts, starts = [0], {1: set(), 2: set()}

    def only(tokens, logits):
        if not tokens:
            prompts[0] += 1
            if prompts[0] == 2:
                logits[:] = -np.inf
                return
        else:
            starts[prompts[0]].add(tokens[0].id)
        kept = logits[777].copy()
        logits[:] = -np.inf
        logits[777] = kept
    fp = _params(wr, 3)
    fp.set_no_timestamps(True); fp.set_max_tokens(6); fp.set_filter_logits_callback(only)
    st = ctx.create_batch_state(1, 4, 1)
    st.set_device_draws(True)
    st.full_batch(fp, [synth_pcm(900, 45 * 16000)])
    assert prompts[0] == 2 and starts == {1: {777}, 2: {0}}, (prompts, starts)
    st.free(); ctx.free()


def test_device_draws_have_the_hosts_log_probabilities(wr, model_path):
    """Where the timestamps outweigh the best text token the text is masked after the row's sum was taken: the drawn timestamp's log-probability
    is relative to that whole sum, with the device's draws as with the host's. The filter sets the rows of the first token: one text token
    and two timestamps, whose sum is known. Bound: the sum's and the exponentials' rounding, 2^-20 of values of about 1."""
    ctx = wr.WhisperContext(model_path("micro.en", decisive=1.0))
    beg = ctx.token_beg()
    x = {777: 1.0, beg + 5: 1.0, beg + 9: 0.9}
    lse = float(np.log(np.sum(np.exp(list(x.values())))))

    seen = set()

    def first(tokens, logits):
        if not tokens:
            logits[:] = -np.inf
            for i, v in x.items():
                logits[i] = v
        else:
            seen.add((tokens[0].id, tokens[0].plog))
    for device in (False, True):
        seen.clear()
        st = ctx.create_batch_state(4, 3, 4)
        st.set_device_draws(device)
        fp = _params(wr, 3)
        fp.set_max_tokens(5); fp.set_filter_logits_callback(first)
        st.full_batch(fp, [synth_pcm(910 + i, 6 * 16000) for i in range(4)])
        assert {t for t, _ in seen} == {beg + 5, beg + 9}, (device, seen)
        for t, p in seen:
            assert abs(p - (x[t] - lse)) < 2.0 ** -20, (device, t, p, x[t] - lse)
        st.free()
    ctx.free()
