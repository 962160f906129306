"""The engine's paths that the serving operators carry (include/moonshine_hip.h): kv_dtype = mxfp4 -- cross K / V in the paged 4-bit
cache, planned, written and attended on the device -- and beam search (msh_set_beam_width: selection and state reordering every step).

mxfp4 is held to the default path's gates (logits max-abs 5e-2, ids wherever the margin exceeds 0.1) against the oracle decoder running on
the SAME quantised keys and values (the engine's own encoder frames, projected and quantised in numpy), so the gate sees every error
but the format's own.  Beam search is held to a numpy search over the engine's own teacher-forced logits: under the uniform kernel set a
row's logits do not depend on what shares its call, so the ids must be equal, not close."""
import os

import numpy as np
import pytest

import serve_ref
import test_gpu_parity as tp
from moonshine_amd import api
from moonshine_amd.hip_api import Engine, MshError
from moonshine_amd.synth import ARCHS, make_audio, synthetic_vocab, write_model_dir
from oracle import host_ref
from oracle import moonshine_ref as ref
from test_gpu_parity import max_decode_len

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def tiled_encoder_mlp(monkeypatch):
    """The encoder's MLP block on the tiled GEMMs: the fused kernel's hidden-64 instance (micro only, reached under uniform kernels) is not
    what these tests are about, and two encodes of one batch must give the same bits here."""
    monkeypatch.setenv("MSH_ENC_MLP", "0")


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).view(np.float32)


def quantised_state(e, w, cfg, clip):
    """The oracle's decoder state on the 4-bit values of the engine's own projected frames."""
    enc = bf16(e.encoder_output(clip))
    st = ref.DecoderState(w, cfg, enc)
    cross = []
    for l in range(cfg.dec_layers):
        p = f"model.decoder.layers.{l}.encoder_attn."
        kv = []
        for name in ("k_proj", "v_proj"):
            x = bf16(enc.astype(np.float64) @ bf16(w[p + name + ".weight"]).astype(np.float64).T)
            x = x.reshape(len(enc), cfg.heads, cfg.head_dim)
            kv.append(np.ascontiguousarray(serve_ref.quantise(x).astype(np.float32).transpose(1, 0, 2)))
        cross.append(tuple(kv))
    st.cross = cross
    return st


def check_logits(e, w, cfg, clips, steps):
    e.set_keep_encoder_output(True)
    e.encode(clips)
    gold, gold_logits = [], []
    for i in range(len(clips)):
        st, toks, lg = quantised_state(e, w, cfg, i), [cfg.bos], []
        for _ in range(steps):
            lg.append(ref.decoder_forward(w, cfg, st, [toks[-1]])[0])
            toks.append(ref.argmax_first(lg[-1]))
        gold.append(toks)
        gold_logits.append(lg)
    toks, logits = e.decode(forced_steps=steps, teacher=np.asarray(gold, np.int32), want_logits=steps)
    worst = 0.0
    for b in range(len(clips)):
        for i in range(steps):
            g = gold_logits[b][i]
            worst = max(worst, float(np.abs(logits[i, b] - g).max()))
            top2 = np.partition(g, -2)[-2:]
            if float(top2[1] - top2[0]) > tp.MARGIN:
                assert toks[b][i + 1] == gold[b][i + 1], (b, i)
    print(f"mxfp4 {cfg.name}: logits max-abs {worst:.4f} over {len(clips)} clips x {steps} steps")
    assert worst <= tp.LOGIT_MAXABS, worst


@pytest.mark.parametrize("arch, lens, steps", [("micro", [16000, 30000, 12345, 9000, 40007], 10), ("micro", [20000], 6), ("tiny", [16000, 33000], 4),
                                               ("base", [24000], 4)])
def test_mxfp4_logits_against_the_oracle_on_the_same_values(tmp_path_factory, arch, lens, steps):
    e, w, cfg = tp._engine(tmp_path_factory, arch, 0)
    e.set_kv_dtype("mxfp4")
    check_logits(e, w, cfg, [make_audio(20 + i, n) for i, n in enumerate(lens)], steps)
    e.close()


def test_mxfp4_switches_and_refusals(tmp_path_factory):
    e, w, cfg = tp._engine(tmp_path_factory, "micro", 0)
    clips = [make_audio(30 + i, 16000 + 1000 * i) for i in range(6)]
    want = e.transcribe_tokens(clips, forced_steps=9)
    e.set_kv_dtype("mxfp4")
    first = e.transcribe_tokens(clips, forced_steps=9)
    assert all(len(t) == 10 for t in first)
    assert e.transcribe_tokens(clips, forced_steps=9) == first           # graph replay, pages planned anew
    other = e.transcribe_tokens(clips[:2] + [make_audio(5, 60000)], forced_steps=9)
    assert len(other) == 3 and e.transcribe_tokens(clips, forced_steps=9) == first
    with pytest.raises(MshError):
        e.set_capture_cross_attention(True)
    e.set_kv_dtype("bf16")
    assert e.transcribe_tokens(clips, forced_steps=9) == want
    e.set_capture_cross_attention(True)
    with pytest.raises(MshError):
        e.set_kv_dtype("mxfp4")
    with pytest.raises(MshError):
        e.set_beam_width(2)
    e.set_capture_cross_attention(False)
    for width, penalty in ((0, 1.0), (17, 1.0), (2, float("nan")), (2, 9.0)):
        with pytest.raises(MshError):
            e.set_beam_width(width, penalty)
    e.set_beam_width(3)
    e.encode(clips)
    with pytest.raises(MshError):
        e.decode(forced_steps=4, want_logits=1)
    with pytest.raises(MshError):
        e.decode(forced_steps=4, teacher=np.ones((6, 5), np.int32))
    with pytest.raises(MshError):
        e.set_capture_cross_attention(True)
    e.set_batches_in_flight(2)
    with pytest.raises(MshError):
        e.set_beam_width(2)
    e.set_batches_in_flight(0)
    e.set_beam_width(1)
    assert e.transcribe_tokens(clips, forced_steps=9) == want
    e.close()


def test_mxfp4_absorbed_form_is_refused(tmp_path_factory):
    e, w, cfg = tp._engine(tmp_path_factory, "tiny", 0)
    e.set_cross_mode("absorbed")
    e.set_kv_dtype("mxfp4")
    with pytest.raises(MshError):
        e.encode([make_audio(1, 16000)])
    e.set_cross_mode("kv")
    e.encode([make_audio(1, 16000)])
    e.close()


def numpy_beams(e, clip, K, steps, eos, penalty):
    """Beam search over the engine's own logits: the clip K times in one batch, each with its hypothesis as the teacher."""
    bos = e.info().bos
    e.set_beam_width(1)
    e.encode([clip] * K)
    hyps, scores, done = [[bos] for _ in range(K)], np.array([0.0] + [-np.inf] * (K - 1), np.float32), np.zeros(K, bool)
    gap = np.inf
    for i in range(steps):
        teacher = np.array([[t if t >= 0 else 0 for t in h] + [0] for h in hyps], np.int32)
        _, logits = e.decode(forced_steps=i + 1, teacher=teacher, want_logits=i + 1)
        s, p, t, f, order = serve_ref.beam_select(logits[i][None], scores[None], done[None], eos)
        # candidates of two beams are sums of different rows: how clearly the order is decided
        (cs, cp), = order
        gap = min([gap] + [abs(a - b) for a, b, x, y in zip(cs, cs[1:], cp, cp[1:]) if x != y])
        hyps = [hyps[p[0, k]] + [-1 if done[p[0, k]] else int(t[0, k])] for k in range(K)]
        scores, done = s[0].astype(np.float32), f[0]
        if done.all():
            break
    lens = [sum(1 for x in h[1:] if x >= 0) for h in hyps]
    best = max(range(K), key=lambda k: (float(scores[k]) / lens[k] ** penalty if lens[k] else -np.inf, -k))
    return [x for x in hyps[best] if x >= 0], gap


@pytest.mark.parametrize("kv_dtype", ["bf16", "mxfp4"])
@pytest.mark.parametrize("K, penalty", [(2, 1.0), (3, 0.0), (5, 2.0)])
def test_beam_search_is_the_search_over_the_engines_logits(tmp_path_factory, K, penalty, kv_dtype):
    """Reference stopping rule (EOS ends a hypothesis, the budget a clip) and forced steps, clips of unlike budgets in one batch."""
    cfg, w, lens, clips = tp.eos_test_weights()
    e, w, cfg = tp._engine(tmp_path_factory, "micro", 39, w)
    e.set_uniform_kernels(True)
    e.set_kv_dtype(kv_dtype)
    e.set_beam_width(K, penalty)
    got = e.transcribe_tokens(clips)
    again = e.transcribe_tokens(clips)
    forced = e.transcribe_tokens(clips[:3], forced_steps=5)
    assert got == again
    ended = checked = 0
    for c, n, g in zip(clips, lens, got):
        want, gap = numpy_beams(e, c, K, max_decode_len(n), cfg.eos, penalty)
        if gap > 1e-5:          # fp32 scores of 64-bit sums: closer candidates may change places
            assert g == want, (n, g, want)
            checked += 1
        ended += g[-1] == cfg.eos
    assert checked >= 6 and (ended >= 1 or penalty > 1)      # (a penalty of 2 favours hypotheses that run to the budget)
    for c, g in zip(clips, forced):
        want, gap = numpy_beams(e, c, K, 5, -1, penalty)
        assert gap <= 1e-5 or g == want
    e.close()


def test_beam_width_one_is_greedy_and_wider_finds_no_worse(tmp_path_factory):
    """Forced steps without a length penalty: the returned hypothesis is at least as likely as the greedy one under the engine's logits."""
    e, w, cfg = tp._engine(tmp_path_factory, "micro", 0)
    e.set_uniform_kernels(True)
    clips = [make_audio(50 + i, 16000 + 3000 * i) for i in range(5)]

    def likelihood(ids):
        e.set_beam_width(1)
        e.encode(clips)
        _, lg = e.decode(forced_steps=7, teacher=np.asarray(ids, np.int32), want_logits=7)
        lg = lg.astype(np.float64)
        lp = lg - (lg.max(-1, keepdims=True) + np.log(np.exp(lg - lg.max(-1, keepdims=True)).sum(-1, keepdims=True)))
        return [sum(lp[i, b, ids[b][i + 1]] for i in range(7)) for b in range(len(clips))]

    greedy = e.transcribe_tokens(clips, forced_steps=7)
    e.set_beam_width(8)
    wide = e.transcribe_tokens(clips, forced_steps=7)
    alone = [e.transcribe_tokens([c], forced_steps=7)[0] for c in clips]
    assert wide == alone
    better = [b - a for a, b in zip(likelihood(greedy), likelihood(wide))]
    assert min(better) > -1e-4, better
    e.set_beam_width(1)
    assert e.transcribe_tokens(clips, forced_steps=7) == greedy
    e.close()


@pytest.mark.parametrize("kv_dtype, mode", [("mxfp4", "kv"), ("bf16", "kv"), ("bf16", "absorbed"), ("fp8", "kv")])
def test_beams_of_real_shapes_in_flight_and_profiled(tmp_path_factory, kv_dtype, mode):
    """The tiny architecture: every cross-attention form under a beam search, lanes against the synchronous call, eager (profiled) against
    replayed steps, batches of changing size."""
    e, w, cfg = tp._engine(tmp_path_factory, "tiny", 0)
    e.set_kv_dtype(kv_dtype)
    e.set_cross_mode(mode)
    e.set_beam_width(4)
    batches = [[make_audio(100 * b + i, 16000 + 2377 * ((7 * i + b) % 11)) for i in range(2 + 9 * b)] for b in range(3)]
    want = [e.transcribe_tokens(c) for c in batches]
    assert all(t[0] == cfg.bos and len(t) > 1 for b in want for t in b)
    e.profile_enable(True)
    assert e.transcribe_tokens(batches[1]) == want[1]
    names = {p["name"] for p in e.profile()}
    assert {"dec_beam_select", "dec_beam_reorder", "dec_beam_advance"} <= names
    assert ("cross_kv4_write" in names) == (kv_dtype == "mxfp4")
    e.profile_enable(False)
    e.set_batches_in_flight(2)
    tickets = [e.submit_transcribe_tokens(c) for c in batches]
    assert [e.wait_tokens(t) for t in tickets] == want
    e.set_batches_in_flight(0)
    e.close()


@pytest.mark.parametrize("beams", [1, 3])
def test_uniform_kernels_give_a_clip_the_same_bits_in_any_batch(tmp_path_factory, beams):
    """mxfp4 under uniform kernels: a clip alone, and in a batch large enough and with a clip long enough that the attention would take
    another form by itself."""
    e, w, cfg = tp._engine(tmp_path_factory, "tiny", 0)
    e.set_uniform_kernels(True)
    e.set_kv_dtype("mxfp4")
    clips = [make_audio(300 + i, 8000 + 512 * (i % 7)) for i in range(150)]
    clips[140] = make_audio(9, 16000 * 24)
    if beams == 1:
        e.encode(clips)
        _, all_logits = e.decode(forced_steps=3, want_logits=3)
        for c in (0, 77, 149):
            e.encode([clips[c]])
            _, logits = e.decode(forced_steps=3, want_logits=3)
            assert np.array_equal(logits[:, 0], all_logits[:, c])
    else:
        e.set_beam_width(beams)
        together = e.transcribe_tokens(clips)
        for c in (0, 77, 140, 149):
            assert e.transcribe_tokens([clips[c]]) == [together[c]]
    e.close()


def test_transcriber_options(tmp_path_factory):
    """kv_dtype = mxfp4, beam_width and length_penalty through the C API: the text is that of the engine's own ids."""
    d = str(tmp_path_factory.mktemp("tiny_model"))
    write_model_dir(d, ARCHS["tiny"], seed=3)
    vocab = synthetic_vocab(ARCHS["tiny"].vocab)
    clips = [make_audio(60 + i, n)[: n // 512 * 512] for i, n in enumerate([16000, 48000, 30720])]
    e = Engine(0)
    e.load_weights_file(os.path.join(d, "model.safetensors"), 0)
    e.set_uniform_kernels(True)
    e.set_kv_dtype("mxfp4")
    e.set_beam_width(3, 0.5)
    want = [host_ref.sanitize_text(host_ref.tokens_to_text(vocab, e.transcribe_tokens([c])[0])) for c in clips]
    e.close()
    base = {"vad_threshold": "0", "kernel_set": "uniform", "kv_dtype": "mxfp4"}
    t = api.Transcriber(d, api.ARCH_TINY, dict(base, beam_width="3", length_penalty="0.5"))
    got = t.transcribe_batch_without_streaming(clips)
    assert [lines[0].text_bytes for lines in got] == want
    assert [t.transcribe_without_streaming(c)[0].text_bytes for c in clips] == want
    t.close()
    for bad in ({"beam_width": "0"}, {"beam_width": "17"}, {"beam_width": "2", "word_timestamps": "true"}, {"word_timestamps": "true"},
                {"cross_attention": "absorbed"}, {"kv_dtype": "fp2"}, {"beam_width": "2", "length_penalty": "100"}):
        with pytest.raises(Exception):
            api.Transcriber(d, api.ARCH_TINY, dict(base, **bad))
